// paged_norm_rotate, hand-written for gfx950: norms of queries and keys a head,
// and their rotation by position.  The host library compiles one entry per
// combination of types, head size, rotated dims and pairing.
#pragma once

#include "ptowsp_blocks_args.h"
#include "ptowsp_numbers.h"

namespace ptowsp {

// ---------------------------------------------------------------------------
// paged_norm_rotate
//
// y = x / sqrt(mean(x^2) + eps) * weight over a head's D dims, in float32; then
// each pair (a, b) of the first R becomes (a cos - b sin, b cos + a sin).  A lane
// holds 2 * P dims, P of them the partners of the others, so that a pair never
// crosses lanes; LANES lanes hold a head, a wave as many heads of one token as
// fit, and goes on with the token's next ones under the same sines.  Its request is
// found 64 steps at a time: two dependent loads for 4096 requests.  Bound by HBM:
// 16384 tokens of 32 + 8 heads of 128 in bf16 (344 MB) 52 us, 6.6 TB/s; 64 tokens by
// latency, 3.9 us.
// ---------------------------------------------------------------------------

// Dims of a lane's piece: a pair's halves shall lie in one lane, so that R's divisors set
// it for the dims that do not turn too.  16384 tokens as above, from memory: R = 128 71 us,
// 96 or 64 78, 36 or 20 132, 4 or 2 117 to 121.
constexpr int rotate_piece(int R) { return R % 16 == 0 ? 8 : R % 8 == 0 ? 4 : R % 4 == 0 ? 2 : 1; }

// ONCE: bytes that the call reads once.  16 of them (a head's dims, side by side in
// a wave) are read without a place in the caches: 16384 tokens of inputs from memory
// take 71 us so and 76 otherwise, of inputs in the caches 52 both.  Other pieces are
// parts of cache lines that another load needs too: float32 heads took 21 us so and 19
// otherwise.
typedef pg_u32 pg_any_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
template <int BYTES, bool ONCE>
__device__ inline void read(void* to, const char* p) {
    if constexpr (ONCE && BYTES == 16) {
        const pg_any_u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const pg_any_u32x4*>(p));
        __builtin_memcpy(to, &w, 16);
    } else {
        __builtin_memcpy(to, p, BYTES);
    }
}
template <int T, int P, bool ONCE = false>
__device__ inline void load_piece(const char* p, float (&y)[P]) {
    if constexpr (T == kF32) {
        read<4 * P, ONCE>(y, p);
    } else if constexpr (T == kF16) {
        _Float16 h[P];
        read<2 * P, ONCE>(h, p);
#pragma unroll
        for (int i = 0; i < P; ++i) y[i] = static_cast<float>(h[i]);
    } else {
        pg_u16 h[P];
        read<2 * P, ONCE>(h, p);
#pragma unroll
        for (int i = 0; i < P; ++i) y[i] = __uint_as_float(static_cast<pg_u32>(h[i]) << 16);
    }
}
template <int T, int P>
__device__ inline void store_piece(char* p, const float (&y)[P]) {
    if constexpr (T == kF32) {
        __builtin_memcpy(p, y, 4 * P);
    } else if constexpr (T == kF16) {
        _Float16 h[P];
#pragma unroll
        for (int i = 0; i < P; ++i) h[i] = static_cast<_Float16>(y[i]);
        __builtin_memcpy(p, h, 2 * P);
    } else {
        __bf16 h[P];
#pragma unroll
        for (int i = 0; i < P; ++i) h[i] = static_cast<__bf16>(y[i]);
        __builtin_memcpy(p, h, 2 * P);
    }
}

// The request whose rows begin last at or ahead of `row`, by 64 steps at a time.
__device__ inline pg_i64 request_of(const RotateArgs& A, pg_i64 row) {
    const int lane = threadIdx.x & 63;
    pg_i64 lo = 0, n = A.batch;  // it is one of lo .. lo + n - 1
    while (n > 1) {
        const pg_i64 step = (n + 63) >> 6, b = lo + lane * step;
        const bool ahead = lane * step < n && A.starts[(lane * step < n ? b : lo) * A.s_starts] <= row;
        const pg_u64 hit = __ballot(ahead);
        const int last = hit ? 63 - __builtin_clzll(hit) : 0;
        lo += last * step;
        n = n - last * step < step ? n - last * step : step;
    }
    return lo;
}

// Where one of a wave's 64 requests starts, and where the next one does.  The search
// takes requests in order and may not meet one that is not, so the first waves look at
// all of them, by loads ahead of the search's; ahead of their own token's the check takes
// 7% of a call of 16384 tokens.
struct Starts {
    int from, to;
    __device__ bool bad(const RotateArgs& A) const { return from < 0 || to < from || to > A.rows; }
};
__device__ inline Starts starts_of(const RotateArgs& A, pg_i64 wave) {
    const pg_i64 b = 64 * wave + (threadIdx.x & 63), at = b < A.batch ? b : A.batch - 1;
    return Starts{A.starts[at * A.s_starts], A.starts[(at + 1) * A.s_starts]};
}

// WT: the type of the weights; QN, KN: whether queries and keys are normalised.
template <int D, int R, int T, int WT, bool QN, bool KN, bool INTER>
struct Rotate {
    static constexpr int P = rotate_piece(R), GROUPS = D / (2 * P), TURN = R / (2 * P);  // groups of 2 P dims; those that turn
    static constexpr int lanes() {
        int n = 1;
        while (n < GROUPS && n < 64) n *= 2;
        return n;
    }
    static constexpr int LANES = lanes(), EACH = (GROUPS + LANES - 1) / LANES, AT_ONCE = 64 / LANES;
    static_assert(D % (2 * P) == 0 && R % (2 * P) == 0 && R >= 2 && R <= D);

    __device__ static int low(int i) { return INTER || i >= TURN ? 2 * P * i : P * i; }
    __device__ static int high(int i) { return INTER || i >= TURN ? 2 * P * i + P : R / 2 + P * i; }

    // Heads first, first + step, ... of the token in `row`, and the order of requests.
    __device__ static void run(const RotateArgs& A, pg_i64 row, int first, int step) {
        const pg_i64 wave = row * step + first;
        const bool looks = 64 * wave < A.batch;
        Starts mine = {0, 0};
        if (looks) mine = starts_of(A, wave);
        turn(A, row, first, step);
        if (looks) {
            bool bad = mine.bad(A);
            for (pg_i64 w = wave + A.rows * step; 64 * w < A.batch; w += A.rows * step) bad |= starts_of(A, w).bad(A);
            if (__ballot(bad)) *A.err = 8;
        }
    }
    __device__ static void turn(const RotateArgs& A, pg_i64 row, int first, int step) {
        const pg_i64 b = request_of(A, row);
        const int s0 = A.starts[b * A.s_starts], s1 = A.starts[(b + 1) * A.s_starts];
        if (row < s0 || row >= s1) return;
        // The token's place among its request's, and its position.
        const pg_i64 place = static_cast<pg_i64>(A.lengths[b * A.s_lengths]) - (s1 - row), pos = place + (A.offsets ? A.offsets[b * A.s_offsets] : 0);
        if (s1 > A.rows || s0 < 0 || place < 0 || pos < 0 || pos >= A.positions) {
            *A.err = 8;
            return;
        }
        const int lane = threadIdx.x & 63, l = lane & (LANES - 1), heads = A.heads[0] + A.heads[1];
        float c[EACH][P], s[EACH][P], w[2][EACH][2][P];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            // Lanes without a group take the last one and write nothing.
            const int i = l + LANES * e < GROUPS ? l + LANES * e : GROUPS - 1, turn = i < TURN ? i : TURN - 1;
            load_piece<kF32, P>(reinterpret_cast<const char*>(A.cos + pos * A.s_cos + P * turn), c[e]);
            load_piece<kF32, P>(reinterpret_cast<const char*>(A.sin + pos * A.s_sin + P * turn), s[e]);
#pragma unroll
            for (int x = 0; x < 2; ++x)
                if (x ? KN : QN) {
                    load_piece<WT, P>(A.weight[x] + low(i) * elem_size(WT), w[x][e][0]);
                    load_piece<WT, P>(A.weight[x] + high(i) * elem_size(WT), w[x][e][1]);
                }
        }
        for (int h0 = first * AT_ONCE; h0 < heads; h0 += step * AT_ONCE) {
            const int h = h0 + lane / LANES, at = h < heads ? h : heads - 1;
            const int key = at >= A.heads[0], hh = key ? at - A.heads[0] : at;
            const char* const x = A.x[key] + (row * A.s_x[key][0] + hh * A.s_x[key][1]) * elem_size(T);
            char* const out = A.out[key] + (row * A.s_out[key][0] + hh * A.s_out[key][1]) * elem_size(T);
            float y[EACH][2][P];
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const bool in = l + LANES * e < GROUPS;
                const int i = in ? l + LANES * e : GROUPS - 1;
                load_piece<T, P, true>(x + low(i) * elem_size(T), y[e][0]);
                load_piece<T, P, true>(x + high(i) * elem_size(T), y[e][1]);
                float part = 0.0f;
#pragma unroll
                for (int k = 0; k < P; ++k) part = __builtin_fmaf(y[e][0][k], y[e][0][k], __builtin_fmaf(y[e][1][k], y[e][1][k], part));
                sum += in ? part : 0.0f;
            }
            if constexpr (QN || KN) {
#pragma unroll
                for (int d = LANES / 2; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
                const float f = 1.0f / sqrtf(sum * (1.0f / D) + A.eps);
                const bool norm = key ? KN : QN;
#pragma unroll
                for (int e = 0; e < EACH; ++e)
#pragma unroll
                    for (int z = 0; z < 2; ++z)
#pragma unroll
                        for (int k = 0; k < P; ++k) {
                            const float weight = QN && KN ? (key ? w[1][e][z][k] : w[0][e][z][k]) : w[KN ? 1 : 0][e][z][k];
                            y[e][z][k] = norm ? y[e][z][k] * f * weight : y[e][z][k];
                        }
            }
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = l + LANES * e;
                if (i < TURN) {
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        // Pair k: of halves (k, k), of neighbours (2k, 2k + 1) in the lane's 2 P dims.
                        float& a = INTER ? y[e][2 * k / P][2 * k % P] : y[e][0][k];
                        float& z = INTER ? y[e][(2 * k + 1) / P][(2 * k + 1) % P] : y[e][1][k];
                        const float a0 = a, z0 = z;
                        a = a0 * c[e][k] - z0 * s[e][k];
                        z = z0 * c[e][k] + a0 * s[e][k];
                    }
                }
                if (i < GROUPS && h < heads) {
                    store_piece<T, P>(out + low(i) * elem_size(T), y[e][0]);
                    store_piece<T, P>(out + high(i) * elem_size(T), y[e][1]);
                }
            }
        }
    }
};

}  // namespace ptowsp
