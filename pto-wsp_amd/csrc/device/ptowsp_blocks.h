// Operators over 8-bit blocks, hand-written for gfx950: e4m3 codes with a
// float32 scale for each block of 128 columns (quantize), and the product of
// such operands (matmul).
#pragma once

#include "ptowsp_blocks_args.h"
#include "ptowsp_numbers.h"

namespace ptowsp {

// ---------------------------------------------------------------------------
// block_quantize
//
// 16 lanes hold the 128 columns of a row's block, eight each: the largest
// finite |x| among them, the scale, the codes.  Weights' blocks have 128 rows as
// well, which a workgroup's 16 groups of lanes share.  A code is the product
// with 1 / scale, rounded as float32 values are.  Infinities and NaN are met
// only where the block's largest bits say so.  Bound by HBM: 16384 rows of 4096 in
// bf16 (203 MB) 32 us, 6.4 TB/s; with NaN tests and clamps on every number 41 us.
// 128-row blocks of the same 37 us, 5.4 TB/s.
// ---------------------------------------------------------------------------

// Columns c .. c + 7 of a row of K; what lies behind K counts as 0.
template <int T>
__device__ inline void row8(const char* row, pg_i64 c, pg_i64 K, Eight<T>& x) {
    if (c + 8 <= K) {
        __builtin_memcpy(x.w, row + c * elem_size(T), 8 * elem_size(T));
        return;
    }
#pragma unroll
    for (int i = 0; i < (T == kF32 ? 8 : 4); ++i) x.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < K) {
            if constexpr (T == kF32) x.w[i] = *reinterpret_cast<const pg_u32*>(row + (c + i) * 4);
            else x.w[i >> 1] |= static_cast<pg_u32>(*reinterpret_cast<const pg_u16*>(row + (c + i) * 2)) << (16 * (i & 1));
        }
}

template <int T>
__device__ inline float number_of(pg_u32 bits) {
    Eight<T> x = {};
    float y[8];
    x.w[0] = bits;
    values8<T>(x, y);
    return y[0];
}

// The largest finite |x| of eight.
template <int T>
__device__ inline float finite8(const Eight<T>& x, float most) {
    float y[8];
    values8<T>(x, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(y[i]);
        if (a < __builtin_inff()) most = fmaxf(most, a);
    }
    return most;
}

// The largest number of this lane and those that differ from it in the bits
// below LANES, without sign.
template <int LANES>
__device__ inline pg_u32 most_bits(pg_u32 x) {
#pragma unroll
    for (int d = LANES / 2; d >= 1; d >>= 1) {
        const pg_u32 y = static_cast<pg_u32>(__shfl_xor(static_cast<int>(x), d, 64));
        x = y > x ? y : x;
    }
    return x;
}

// FINITE: all numbers of the block are, and none is beyond the largest code by more
// than a few roundings of float32, which round away again.
template <int T, bool FINITE>
__device__ inline pg_u32 codes8(const Eight<T>& x, float inverse, pg_u32& hi) {
    float y[8];
    values8<T>(x, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= inverse;
    hi = encode4<kE4M3, FINITE>(y + 4);
    return encode4<kE4M3, FINITE>(y);
}

__device__ inline void put8(char* row, pg_i64 c, pg_i64 K, pg_u32 lo, pg_u32 hi) {
    if (c + 8 <= K) {
        const pg_u32x2 w = {lo, hi};
        __builtin_memcpy(row + c, &w, 8);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < K) row[c + i] = static_cast<char>((i < 4 ? lo : hi) >> (8 * (i & 3)));
}

// Blocks of one row, U for each 16 lanes.
template <int T, int U>
__device__ inline void quantize_rows(const QuantizeArgs& A) {
    const pg_u32 first = blockIdx.x * (16 * U) + (threadIdx.x >> 4);
    const int l = threadIdx.x & 15;
    Eight<T> x[U];
    pg_i64 row[U];
    pg_u32 block[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const pg_u32 i = first + 16 * u;
        in[u] = i < A.many;
        const pg_u32 at = in[u] ? i : A.many - 1, r = at / A.blocks;
        row[u] = r;
        block[u] = at - r * A.blocks;
        row8<T>(A.x + row[u] * A.s_x * elem_size(T), block[u] * kScaleBlock + 8 * l, A.cols, x[u]);
    }
    constexpr pg_u32 kInf = T == kF32 ? 0x7F800000u : T == kF16 ? 0x7C00u : 0x7F80u;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        pg_u32 bits = most8<T>(x[u], 0);
        if constexpr (T != kF32) bits = (bits & 0xFFFFu) > bits >> 16 ? bits & 0xFFFFu : bits >> 16;
        bits = most_bits<16>(bits);
        float most = number_of<T>(bits);
        const bool finite = __ballot(bits >= kInf) == 0;
        if (!finite) most = __uint_as_float(most_bits<16>(__float_as_uint(finite8<T>(x[u], 0.0f))));
        const float scale = fmaxf(most / 448.0f, 0x1p-126f), inverse = 1.0f / scale;
        pg_u32 lo, hi;
        if (finite) lo = codes8<T, true>(x[u], inverse, hi);
        else lo = codes8<T, false>(x[u], inverse, hi);
        if (in[u]) {
            put8(A.codes + row[u] * A.s_codes, block[u] * kScaleBlock + 8 * l, A.cols, lo, hi);
            if (l == 0) A.scales[row[u] * A.s_scales[0] + block[u] * A.s_scales[1]] = scale;
        }
    }
}

// A block of 128 rows, for a workgroup of 256 threads.
template <int T>
__device__ inline void quantize_squares(const QuantizeArgs& A) {
    __shared__ pg_u32 most4[4];
    const pg_u32 strip = blockIdx.x / A.blocks, block = blockIdx.x - strip * A.blocks;
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const pg_i64 r0 = static_cast<pg_i64>(strip) * kScaleBlock, c = static_cast<pg_i64>(block) * kScaleBlock + 8 * l;
    Eight<T> x[8];
    float fine = 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const pg_i64 r = r0 + g + 16 * u;  // rows behind the last one repeat it
        row8<T>(A.x + (r < A.rows ? r : A.rows - 1) * A.s_x * elem_size(T), c, A.cols, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) fine = finite8<T>(x[u], fine);
    const pg_u32 most = most_bits<64>(__float_as_uint(fine));
    if ((threadIdx.x & 63) == 0) most4[threadIdx.x >> 6] = most;
    __syncthreads();
    pg_u32 all = most4[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) all = most4[w] > all ? most4[w] : all;
    const float scale = fmaxf(__uint_as_float(all) / 448.0f, 0x1p-126f), inverse = 1.0f / scale;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const pg_i64 r = r0 + g + 16 * u;
        pg_u32 hi;
        const pg_u32 lo = codes8<T, false>(x[u], inverse, hi);
        if (r < A.rows) put8(A.codes + r * A.s_codes, c, A.cols, lo, hi);
    }
    if (threadIdx.x == 0) A.scales[strip * A.s_scales[0] + block * A.s_scales[1]] = scale;
}

// ---------------------------------------------------------------------------
// block_matmul
//
// A stage is one block of K, 128 codes.  The sum of its products enters the
// accumulators by a multiplication with the block's two scales, in float32.  The
// weights are the MFMA's rows and the activations its columns, so that a lane's
// numbers belong to one row of `a`, and to four neighbouring columns of the
// result.
//
// For 16-bit results v_mfma_f32_16x16x128 takes the codes as they are.  It adds
// products eight by eight, and cuts them at 2^-13 of the largest of the eight
// (found with powers of two at every place; e4m3's older MFMAs do the same); the
// eights it adds as float32 numbers.  For random rows that is 1.5e-5 of the
// result, a tenth of what rounding to f16 costs and a hundredth of bf16's, but 25
// times float32's: for float32 results the codes become bf16 values, exactly, for
// v_mfma_f32_16x16x32, at half the rate, whose products and sums are float32's.
//
// The host chooses the tile and the shares of K by a fitted cost (BlockStream for up
// to 16 rows).  Many rows are bound by the clock that the card's power leaves and by
// instructions beside the MFMAs: 8192 x 6144 x 4096 to bf16 220 us, 1.87 PFLOP/s (10%
// less with all codes zero).  Few rows by the way of the weights through the ring, 32
// stages one behind the other: 64 x 6144 x 4096 (27 MB) 13.3 us, 2.0 TB/s; deeper rings,
// wider tiles, shares of K and an order of stages of its own for each workgroup gain
// nothing.  The stream takes 8.5 us for one row of these weights, 12.4 for 16.
// ---------------------------------------------------------------------------

typedef int pg_i32x8 __attribute__((ext_vector_type(8)));

// A scale as factor * 2^(power - 127), each with half of its exponent.  The power goes to
// the codes, in the conversion or the MFMA: so neither a block's sum (0, or 2^-18 to 2^25
// and its sign, times two powers) nor the product of two factors leaves float32 where the
// result does not, and a sum of 0 adds 0; nothing else is rounded than in a product of
// the two scales, which alone may lie below 2^-126 or beyond 2^128.  Factors are below
// 2^64, those of normal numbers 2^-63 and above; infinities and NaN are factors.  Against
// that product 8192 x 6144 x 4096 takes 2% longer to bf16 and to float32, 1024 rows 4%, 64
// rows 3%; a branch for such products alone took as long or spilled registers.
__device__ inline int power_of(float scale) { return static_cast<int>((__float_as_uint(scale) >> 24 & 0x7Fu) + 64u); }
__device__ inline float factor_of(float scale, int power) { return scale * __uint_as_float(static_cast<pg_u32>(254 - power) << 23); }
struct Halves {
    float factor;
    int power;  // 64 .. 191
    __device__ explicit Halves(float scale) : power(power_of(scale)) { factor = factor_of(scale, power); }
    Halves() = default;
};
// Of a scale that all lanes have, in vector registers as the others: the MFMA takes its
// powers from no other ones, which not every compiler knows.
__device__ inline Halves uniform_halves(float scale) {
    asm("" : "+v"(scale));
    return Halves(scale);
}

// A lane's 32 codes of a row in a stage, as they are or WIDE, times 2^(power - 127) as bf16.
template <bool WIDE>
struct Codes32 {
    pg_u32x4 w[WIDE ? 4 : 2];
    __device__ Codes32(pg_u32x4 x, pg_u32x4 y, int power) {
        if constexpr (WIDE) {
            const pg_u32x4 in[2] = {x, y};
            const float f = __uint_as_float(static_cast<pg_u32>(power) << 23);
            auto two = [&](pg_u32 w, auto hi) { return __builtin_bit_cast(pg_u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, f, decltype(hi)::value)); };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const pg_u32 lo = in[i >> 1][2 * (i & 1)], hi = in[i >> 1][2 * (i & 1) + 1];
                w[i] = pg_u32x4{two(lo, Flag<false>()), two(lo, Flag<true>()), two(hi, Flag<false>()), two(hi, Flag<true>())};
            }
        } else {
            w[0] = x;
            w[1] = y;
        }
    }
    Codes32() = default;
};

// pa, pb: powers of codes that are as they are.
template <bool WIDE>
__device__ inline pg_f32x4 stage_sum(const Codes32<WIDE>& a, const Codes32<WIDE>& b, int pa, int pb) {
    pg_f32x4 c = {0, 0, 0, 0};
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf8, a.w[i]), __builtin_bit_cast(pg_bf8, b.w[i]), c, 0, 0, 0);
        return c;
    } else {
        struct Pair {
            pg_u32x4 w[2];
        };
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(pg_i32x8, Pair{{a.w[0], a.w[1]}}), __builtin_bit_cast(pg_i32x8, Pair{{b.w[0], b.w[1]}}), c,
                                                                0, 0, 0, pa, 0, pb);
    }
}

// Codes k .. k + 15 of a row of K, at any address; what lies behind K is 0.
__device__ inline pg_u32x4 codes16(const char* row, pg_i64 k, pg_i64 K) {
    pg_u32x4 w = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&w, row + k, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (k + i < K) w[i >> 2] |= static_cast<pg_u32>(static_cast<pg_u8>(row[k + i])) << (8 * (i & 3));
    }
    return w;
}

// Columns n .. of a row of N results.
template <int T, bool INSIDE, int MANY>
__device__ inline void put_row(char* out, pg_i64 n, pg_i64 N, const float (&y)[MANY]) {
    char* const p = out + n * elem_size(T);
    if (INSIDE || n + MANY <= N) {
        if constexpr (T == kF32) {
            __builtin_memcpy(p, y, 4 * MANY);
        } else {
            pg_u32 w[MANY / 2];
#pragma unroll
            for (int i = 0; i < MANY / 2; ++i) {
                if constexpr (T == kF16) w[i] = __builtin_bit_cast(pg_u32, (pg_h2{static_cast<_Float16>(y[2 * i]), static_cast<_Float16>(y[2 * i + 1])}));
                else w[i] = __builtin_bit_cast(pg_u32, __builtin_convertvector((pg_f32x2{y[2 * i], y[2 * i + 1]}), pg_bf2));
            }
            __builtin_memcpy(p, w, 2 * MANY);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < MANY; ++i)
        if (n + i < N) store_elem<T>(p + i * elem_size(T), y[i]);
}
template <int T, bool INSIDE>
__device__ inline void put4(char* out, pg_i64 n, pg_i64 N, pg_f32x4 x) {
    put_row<T, INSIDE, 4>(out, n, N, {x[0], x[1], x[2], x[3]});
}
template <int T, bool INSIDE>
__device__ inline void put8(char* out, pg_i64 n, pg_i64 N, pg_f32x4 x, pg_f32x4 y) {
    put_row<T, INSIDE, 8>(out, n, N, {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
}

// Raw buffer descriptor for p (no range check: offsets are bounded on the host).
__device__ inline pg_u32x4 buffer_at(const void* p) {
    const pg_u64 a = reinterpret_cast<pg_u64>(p);
    return pg_u32x4{static_cast<pg_u32>(__builtin_amdgcn_readfirstlane(static_cast<int>(a))),
                    static_cast<pg_u32>(__builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32))) & 0xFFFFu, 0xFFFFFFFFu, 0x00020000u};
}
// 16 (or 4) bytes per lane from a buffer into LDS at `lds` + 16 (or 4) * lane.
// In inline asm: the compiler would wait for it ahead of every LDS read.  The
// caller waits with landed_and_read() and a barrier before it reads them.
__device__ inline void to_lds16(pg_u32x4 buffer, int voff, int soff, pg_u32 lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(buffer), "s"(soff), "s"(lds)
                 : "memory", "m0");
}
__device__ inline void to_lds4(pg_u32x4 buffer, int voff, int soff, pg_u32 lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(buffer), "s"(soff), "s"(lds)
                 : "memory", "m0");
}
// All but this wave's last N loads have landed, and its reads of LDS have ended.
template <int N>
__device__ inline void landed_and_read() {
    static_assert(N < 64);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// The same but for the last `many` stages, MOST at most, of LOADS loads each (the
// last of MOST: LAST).
template <int MOST, int LOADS, int LAST = LOADS>
__device__ inline void landed_of(int many) {
    if constexpr (MOST == 0) {
        landed_and_read<0>();
    } else {
        if (many >= MOST) landed_and_read<(MOST - 1) * LOADS + LAST>();
        else landed_of<MOST - 1, LOADS>(many);
    }
}
__device__ inline void meet() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <int V>
struct Int {
    static constexpr int value = V;
};

// BM x BN results for a workgroup of WM x WN waves; a ring of NS stages of K in LDS.
// The loads of a stage to come are spread among the MFMAs of this one, and a block's
// scales enter two MFMAs behind its sum.
// DIRECT: rows, their distances and K are multiples of 16 bytes, and codes go from
// memory straight to LDS; otherwise through registers, at any address.
template <int BM, int BN, int WM, int WN, int NS, bool DIRECT, int T>
struct BlockGemm {
    static constexpr bool WIDE = T == kF32;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
    static constexpr int PIECES = (BM + BN) * 8 / THREADS, AP = BM * 8 / THREADS;  // 16-byte pieces of a stage that a thread loads, and of a's
    static constexpr bool PAIRS = TN % 32 == 0;
    static constexpr int SM = BM < 64 ? 64 : BM, SLOADS = (SM / 64 + WAVES - 1) / WAVES, LOADS = PIECES + SLOADS;
    static constexpr int STAGE = (BM + BN) * 128 + SM * 4;
    static_assert(FM > 1 && kScaleBlock % TN == 0 && (BM + BN) * 8 % THREADS == 0 && BM * 8 % THREADS == 0);

    // Of each stage rows of 128 codes, those of `a` first, then the scales of a's
    // rows.  Piece c of row r lies at c ^ key(r): the rows of an operand's read meet
    // in no bank.
    struct Shared {
        alignas(1024) char bytes[(DIRECT ? NS : 1) * STAGE];
    };

    __device__ static int key_a(int r) { return r & 7; }
    __device__ static int key_b(int r) { return PAIRS ? (r & 3) | (r >> 1 & 4) : r & 7; }

    struct Place {
        pg_i64 m0, n0;
        int split;
    };
    // Workgroups take turns on the 8 XCDs: each gets a run of neighbouring tiles, 8
    // rows of tiles deep.
    __device__ static Place place(const MatmulArgs& A) {
        const int all = A.tiles_m * A.tiles_n, split = blockIdx.x / all, id = blockIdx.x - split * all, xcd = id & 7;
        const int t = (all >> 3) * xcd + (xcd < (all & 7) ? xcd : all & 7) + (id >> 3);
        const int deep = 8 * A.tiles_n, strip = t / deep, in = t - strip * deep, rows = A.tiles_m - 8 * strip < 8 ? A.tiles_m - 8 * strip : 8;
        const int n = in / rows;
        return Place{static_cast<pg_i64>(8 * strip + in - n * rows) * BM, static_cast<pg_i64>(n) * BN, split};
    }

    __device__ static void run(const MatmulArgs& A, Shared& sh) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave - wm * WN;
        const int c = lane & 15, g = lane >> 4;
        const Place at = place(A);
        const int rows = A.M - at.m0 < BM ? static_cast<int>(A.M - at.m0) : BM, cols = A.N - at.n0 < BN ? static_cast<int>(A.N - at.n0) : BN;
        pg_f32x4 acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = pg_f32x4{0, 0, 0, 0};
        const pg_i64 strip = (at.n0 + wn * TN) / kScaleBlock, strips = (A.N + kScaleBlock - 1) / kScaleBlock;
        // The split's stages, and its codes of a row.
        const int first = static_cast<int>(static_cast<pg_i64>(A.stages) * at.split / A.splits);
        const int stages = static_cast<int>(static_cast<pg_i64>(A.stages) * (at.split + 1) / A.splits) - first;
        const pg_i64 k0 = static_cast<pg_i64>(first) * kScaleBlock, K = A.K - k0 < static_cast<pg_i64>(stages) * kScaleBlock ? A.K - k0 : static_cast<pg_i64>(stages) * kScaleBlock;
        const char* const a0 = A.a + at.m0 * A.s_a + k0;
        const char* const b0 = A.b + at.n0 * A.s_b + k0;
        const float* const as0 = A.a_scale + at.m0 * A.s_as[0] + first * A.s_as[1];
        const pg_u32x4 buf_a = buffer_at(a0), buf_b = buffer_at(b0), buf_s = buffer_at(as0);
        const pg_u32 lds = static_cast<pg_u32>(reinterpret_cast<pg_u64>((const __attribute__((address_space(3))) void*)sh.bytes));
        const int tail = static_cast<int>(K - static_cast<pg_i64>(stages - 1) * kScaleBlock);  // codes of the last stage
        // A thread's pieces: slot i & 7 of row i >> 3 holds the piece (i ^ row) & 7.
        int voff[PIECES], soff_s[SLOADS];
        pg_i64 far[PIECES];  // the same without a limit
        auto piece_row = [&](int p) { return static_cast<int>(threadIdx.x + THREADS * p) >> 3; };
        const int slot = static_cast<int>(threadIdx.x) & 7, row8 = static_cast<int>(threadIdx.x) >> 3;
        const int col[2] = {(slot ^ key_a(row8)) * 16, (slot ^ key_b(row8)) * 16};  // first codes of its pieces of a, of b
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int r = piece_row(p);
            // Rows behind the last one repeat it; their results are not stored.
            far[p] = r < BM ? (r < rows ? r : rows - 1) * A.s_a : (r - BM < cols ? r - BM : cols - 1) * A.s_b;
            voff[p] = static_cast<int>(far[p]) + col[p >= AP];
        }
#pragma unroll
        for (int p = 0; p < SLOADS; ++p) {
            const int r = (wave + WAVES * p) % (SM / 64) * 64 + lane;
            soff_s[p] = static_cast<int>((r < rows ? r : rows - 1) * A.s_as[0]) * 4;
        }
        // The p-th of a wave's loads of stage s, into a place of the ring.
        auto load = [&](int s, int slot, int p, const int (&back)[2]) {
            const pg_u32 base = lds + slot * STAGE;
            if (p < PIECES) {
                to_lds16(p < AP ? buf_a : buf_b, voff[p < PIECES ? p : 0] - back[p >= AP], s * kScaleBlock, base + (wave * 64 + THREADS * p) * 16);
            } else {
                const int q = p - PIECES;
                to_lds4(buf_s, soff_s[q], static_cast<int>(s * A.s_as[1]) * 4, base + (BM + BN) * 128 + (wave + WAVES * q) % (SM / 64) * 256);
            }
        };
        // The scale of the weights' block, through the scalar cache, a stage ahead of its use.
        const auto* const bs = reinterpret_cast<const __attribute__((address_space(4))) float*>(
            reinterpret_cast<pg_u64>(A.b_scale + (strip < strips ? strip : strips - 1) * A.s_bs[0] + first * A.s_bs[1]));
        auto weight_scale = [&](int s) { return bs[(s < stages ? s : stages - 1) * A.s_bs[1]]; };
        // Where this lane's pieces of a row lie, in every 16 rows alike.  Its four numbers
        // of columns 16j .. and of 16 (j + 1) .. shall be neighbours in the result, so the
        // MFMAs' rows 4g + e of both are columns 8g + e and 8g + 4 + e.
        const int rb = PAIRS ? 8 * (c >> 2) + (c & 3) : c;
        int piece_a[2], piece_b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            piece_a[h] = c * 128 + ((g + 4 * h) ^ key_a(c)) * 16;
            piece_b[h] = rb * 128 + ((g + 4 * h) ^ key_b(rb)) * 16;
        }
        auto column = [](int j) { return PAIRS ? 32 * (j >> 1) + 4 * (j & 1) : 16 * j; };
        const int arow = wm * TM * 128, brow = (BM + wn * TN) * 128, srow = (BM + BN) * 128 + (wm * TM + c) * 4;
        // What the wave has read of a stage: its columns, and the next 16 rows.
        Codes32<WIDE> b[FN];
        pg_u32x4 raw[2];
        Halves weight, row;  // of the stage's weights, and of the next 16 rows
        float scale;         // of the 16 rows behind those, read ahead of their codes
        auto read = [&](const char* p) { return *reinterpret_cast<const pg_u32x4*>(p); };
        auto read_rows = [&](const char* stage, int i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) raw[h] = read(stage + arow + i * 2048 + piece_a[h]);
        };
        auto scale_at = [&](const char* stage, int i) { return *reinterpret_cast<const float*>(stage + srow + 64 * i); };
        auto read_column = [&](const char* stage, int j, int limit, int power) {
            pg_u32x4 w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[h] = read(stage + brow + column(j) * 128 + piece_b[h]);
                if (limit) {  // the stage's codes
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[h][e] = 64 * h + 16 * g < limit ? w[h][e] : 0;
                }
            }
            b[j] = Codes32<WIDE>(w[0], w[1], power);
        };
        // The MFMAs of stage s, of which the columns and the first rows have been read.
        // A sum is used two MFMAs later.  At POINT the stage's last rows have been read,
        // and the workgroup meets: the next stage has landed, and this one's place is
        // free.  Its columns follow those of this stage as their last MFMAs begin.  The
        // loads are spread among the MFMAs, since each holds up the wave until it has
        // left: EARLY of them behind POINT, a stage ahead of the others.  The order is
        // kept as it stands here.
        // KIND: 3 all stages up to s + NS are there to load; 2 none behind s + NS - 1; 1
        // nothing is left to load; 0 the last stage.
        constexpr int MANY = FM * FN, LAG = MANY > 2 ? 2 : MANY - 1;
        constexpr int POINT = (FM - 2) * FN + FN / 2, EARLY = LOADS * (MANY - POINT) / MANY;
        int s = 0, ring = 0;
        // TOGETHER: the next stage's first scales are read with its first rows, all ahead of an
        // MFMA that waits for reads, instead of at POINT: 64 rows of 6144 x 4096 gain 3%, 128
        // rows 3%, 8192 rows to float32 2%; 1024 rows to bf16 would lose 2%.
        constexpr bool TOGETHER = WIDE || FN <= 2;
        // next: the next stage's scale of the weights, which has been loaded.
        auto body = [&](auto kind, float next, const int (&back1)[2], const int (&back2)[2]) {
            constexpr int KIND = decltype(kind)::value;
            const int after = ring == NS - 1 ? 0 : ring + 1, before = ring == 0 ? NS - 1 : ring - 1;
            const char* const stage = sh.bytes + ring * STAGE;
            const char* const behind = sh.bytes + after * STAGE;
            const int limit = KIND == 3 ? 0 : s + 2 == stages ? tail : kScaleBlock;
            pg_f32x4 y[LAG + 1];
            float f[2];
            int power = 0;
            Codes32<WIDE> a;
            Halves follows;
            float later;
            auto add = [&](int k) {
                const int i = k / FN, j = k - i * FN;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(y[k % (LAG + 1)][e], f[i & 1], acc[i][j][e]);
            };
#pragma unroll
            for (int k = 0; k < MANY; ++k) {
                const int i = k / FN, j = k - i * FN;
                if (j == 0) {
                    f[i & 1] = row.factor * weight.factor;
                    power = row.power;
                    a = Codes32<WIDE>(raw[0], raw[1], power);
                    if (WIDE && KIND > 0 && i == FM - 1) follows = uniform_halves(next);
                    if (i + 1 < FM) read_rows(stage, i + 1);
                    else if (KIND > 0) read_rows(behind, 0);
                    if (i + 1 < FM) row = Halves(scale);
                    if (i + 2 < FM) scale = scale_at(stage, i + 2);
                    else if (KIND > 0 && i == FM - 1) later = scale_at(behind, 1);
                    if (TOGETHER && KIND > 0 && i == FM - 1) {
                        scale = scale_at(behind, 0);
                        __builtin_amdgcn_sched_barrier(0);  // these loads ahead of the MFMA's wait
                    }
                }
                y[k % (LAG + 1)] = stage_sum<WIDE>(b[j], a, weight.power, power);
                if constexpr (KIND > 0) {
                    if (KIND > 1 && k < POINT) {
#pragma unroll
                        for (int p = EARLY + k * (LOADS - EARLY) / POINT; p < EARLY + (k + 1) * (LOADS - EARLY) / POINT; ++p) load(s + NS - 1, before, p, back1);
                    }
                    if (k == POINT) {
                        if (KIND > 1 && POINT == 0) {
#pragma unroll
                            for (int p = EARLY; p < LOADS; ++p) load(s + NS - 1, before, p, back1);
                        }
                        if (KIND > 1 || NS == 2) landed_and_read<(NS - 2) * LOADS>();
                        else landed_of<NS - 2, LOADS>(stages - s - 2);
                        meet();
                        if (!TOGETHER) scale = scale_at(behind, 0);
                    }
                    if (KIND > 2 && k >= POINT) {
#pragma unroll
                        for (int p = (k - POINT) * EARLY / (MANY - POINT); p < (k - POINT + 1) * EARLY / (MANY - POINT); ++p) load(s + NS, ring, p, back2);
                    }
                    if (i == FM - 1) read_column(behind, j, limit, follows.power);
                }
                if (k >= LAG) add(k - LAG);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int k = MANY - LAG; k < MANY; ++k) add(k);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (KIND > 0) {
                weight = WIDE ? follows : uniform_halves(next);
                row = Halves(scale);
                scale = later;
            }
            ring = after;
            ++s;
        };
        auto begin = [&](int limit, float weights) {
            weight = uniform_halves(weights);
            row = Halves(scale_at(sh.bytes, 0));
            scale = scale_at(sh.bytes, 1);
            read_rows(sh.bytes, 0);
#pragma unroll
            for (int j = 0; j < FN; ++j) read_column(sh.bytes, j, limit, weight.power);
        };
        if constexpr (DIRECT) {
            // Pieces behind K repeat the row's last one; their weights are cleared where
            // they are read.
            const int none[2] = {0, 0}, back[2] = {col[0] > tail - 16 ? col[0] - (tail - 16) : 0, col[1] > tail - 16 ? col[1] - (tail - 16) : 0};
            auto back_of = [&](int stage, int (&x)[2]) {
                x[0] = stage == stages - 1 ? back[0] : 0;
                x[1] = stage == stages - 1 ? back[1] : 0;
            };
            int now[2];
#pragma unroll
            for (int q = 0; q < NS; ++q) {
                back_of(q, now);
                if (q < stages)
#pragma unroll
                    for (int p = 0; p < (q < NS - 1 ? LOADS : EARLY); ++p) load(q, q, p, now);
            }
            landed_of<NS - 1, LOADS, EARLY>(stages - 1);
            meet();
            begin(stages == 1 ? tail : kScaleBlock, weight_scale(0));
            float next = weight_scale(1), coming;
            while (s + NS < stages) {
                coming = weight_scale(s + 2);
                back_of(s + NS, now);
                body(Int<3>(), next, none, now);
                next = coming;
            }
            if (s + NS == stages) {
                coming = weight_scale(s + 2);
                body(Int<2>(), next, back, none);
                next = coming;
            }
            while (s + 1 < stages) {
                coming = weight_scale(s + 2);
                body(Int<1>(), next, none, none);
                next = coming;
            }
            body(Int<0>(), next, none, none);
        } else {
            pg_u32x4 w[PIECES];
            auto fetch = [&](int s) {
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
                    w[p] = codes16((p < AP ? a0 : b0) + far[p], static_cast<pg_i64>(s) * kScaleBlock + col[p >= AP], K);
            };
            fetch(0);
            for (int t = 0; t < stages; ++t) {
                __syncthreads();
#pragma unroll
                for (int p = 0; p < PIECES; ++p) *reinterpret_cast<pg_u32x4*>(sh.bytes + (threadIdx.x + THREADS * p) * 16) = w[p];
                for (int r = threadIdx.x; r < BM; r += THREADS)
                    reinterpret_cast<float*>(sh.bytes + (BM + BN) * 128)[r] = as0[(r < rows ? r : rows - 1) * A.s_as[0] + t * A.s_as[1]];
                __syncthreads();
                if (t + 1 < stages) fetch(t + 1);
                const int none[2] = {0, 0};
                begin(0, weight_scale(t));
                body(Int<0>(), 0.0f, none, none);
                ring = 0;
            }
        }
        auto store = [&](auto whole, auto type, char* to, pg_i64 stride) {
            constexpr bool INSIDE = decltype(whole)::value;
            constexpr int OT = decltype(type)::value;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int r = wm * TM + 16 * i + c;
                if (!INSIDE && r >= rows) continue;
                char* const out = to + (at.m0 + r) * stride * elem_size(OT);
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    if constexpr (PAIRS) {
                        if (j % 2 == 0) put8<OT, INSIDE>(out, at.n0 + wn * TN + 16 * j + 8 * g, A.N, acc[i][j], acc[i][j + 1]);
                    } else {
                        put4<OT, INSIDE>(out, at.n0 + wn * TN + 16 * j + 4 * g, A.N, acc[i][j]);
                    }
                }
            }
        };
        if (A.splits > 1) store(Flag<false>(), Int<kF32>(), reinterpret_cast<char*>(A.parts + at.split * A.M * A.N), A.N);
        else if (rows == BM && cols == BN) store(Flag<true>(), Int<T>(), A.out, A.s_out);
        else store(Flag<false>(), Int<T>(), A.out, A.s_out);
    }
};

// Up to 16 rows of a: the weights are the work, and each is used once, so that they
// go from memory straight to the MFMAs' registers.  A workgroup has 16 columns; its
// waves share the stages of K, and their sums are added in LDS, in order.
template <int WAVES, bool DIRECT, int T>
struct BlockStream {
    static constexpr bool WIDE = T == kF32;
    struct Shared {
        pg_f32x4 sums[WAVES][64];
    };
    struct Stage {
        pg_u32x4 a[2], b[2];
        float scale, weight;
    };

    __device__ static void run(const MatmulArgs& A, Shared& sh) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
        const int split = blockIdx.x / A.tiles_n, tile = blockIdx.x - split * A.tiles_n;
        const pg_i64 n0 = static_cast<pg_i64>(tile) * 16;
        const int shares = A.splits * WAVES, share = split * WAVES + wave;
        int s = static_cast<int>(static_cast<pg_i64>(A.stages) * share / shares);
        const int end = static_cast<int>(static_cast<pg_i64>(A.stages) * (share + 1) / shares);
        // Rows and columns behind the last one repeat it; their results are not stored.
        const pg_i64 row = c < A.M ? c : A.M - 1, col = n0 + c < A.N ? n0 + c : A.N - 1;
        const char* const a = A.a + row * A.s_a;
        const char* const b = A.b + col * A.s_b;
        const float* const as = A.a_scale + row * A.s_as[0];
        const float* const bs = A.b_scale + n0 / kScaleBlock * A.s_bs[0];
        auto load = [&](int t, Stage& x) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const pg_i64 k = static_cast<pg_i64>(t) * kScaleBlock + 64 * h + 16 * g;
                if constexpr (DIRECT) {
                    // Pieces behind K repeat the row's last one; their weights are cleared in add().
                    const pg_i64 at = k < A.K ? k : A.K - 16;
                    x.a[h] = *reinterpret_cast<const pg_u32x4*>(a + at);
                    x.b[h] = *reinterpret_cast<const pg_u32x4*>(b + at);
                } else {
                    x.a[h] = codes16(a, k, A.K);
                    x.b[h] = codes16(b, k, A.K);
                }
            }
            x.scale = as[t * A.s_as[1]];
            x.weight = bs[t * A.s_bs[1]];
        };
        pg_f32x4 acc = {0, 0, 0, 0};
        auto add = [&](int t, Stage& x) {
            if (DIRECT && static_cast<pg_i64>(t + 1) * kScaleBlock > A.K) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool in = static_cast<pg_i64>(t) * kScaleBlock + 64 * h + 16 * g < A.K;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x.b[h][e] = in ? x.b[h][e] : 0;
                }
            }
            const Halves row(x.scale), weight = uniform_halves(x.weight);
            const pg_f32x4 y = stage_sum<WIDE>(Codes32<WIDE>(x.b[0], x.b[1], weight.power), Codes32<WIDE>(x.a[0], x.a[1], row.power), weight.power, row.power);
            const float f = row.factor * weight.factor;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(y[e], f, acc[e]);
        };
        // The stages ahead are under way during one.
        constexpr int AHEAD = 4;
        Stage x[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD - 1; ++q)
            if (s + q < end) load(s + q, x[q]);
        while (s < end) {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                if (s + AHEAD - 1 < end) load(s + AHEAD - 1, x[(q + AHEAD - 1) % AHEAD]);
                if (s < end) add(s, x[q]);
                ++s;
            }
        }
        sh.sums[wave][lane] = acc;
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) acc += sh.sums[w][lane];
        if (c >= A.M) return;
        if (A.splits == 1) put4<T, false>(A.out + c * A.s_out * elem_size(T), n0 + 4 * g, A.N, acc);
        else put4<kF32, false>(reinterpret_cast<char*>(A.parts + (split * A.M + c) * A.N), n0 + 4 * g, A.N, acc);
    }
};

// The sums of the splits, in order.  Four columns a thread.
template <int T>
__device__ inline void join_splits(const MatmulArgs& A) {
    const pg_i64 fours = (A.N + 3) / 4, item = static_cast<pg_i64>(blockIdx.x) * blockDim.x + threadIdx.x, m = item / fours, n = 4 * (item - m * fours);
    if (m >= A.M) return;
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < A.splits; ++s) {
        const float* const p = A.parts + (s * A.M + m) * A.N + n;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] += p[n + e < A.N ? e : 0];
    }
    put_row<T, false, 4>(A.out + m * A.s_out * elem_size(T), n, A.N, y);
}

}  // namespace ptowsp
