// Operators over a paged KV cache held in 8 bits, hand-written for gfx950:
// block tables and slot maps (plan), quantising writes (store) and causal
// grouped-query attention (attend).  The host library compiles one entry per
// combination of types, head size, page size and group.
#pragma once

#include "ptowsp_paged_args.h"

namespace ptowsp {

typedef long long pg_i64;
typedef unsigned int pg_u32;
typedef unsigned long long pg_u64;
typedef unsigned short pg_u16;
typedef unsigned char pg_u8;
typedef pg_u32 pg_u32x2 __attribute__((ext_vector_type(2)));
typedef pg_u32 pg_u32x4 __attribute__((ext_vector_type(4)));
typedef float pg_f32x2 __attribute__((ext_vector_type(2)));
typedef float pg_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pg_bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef float pg_f32x16 __attribute__((ext_vector_type(16)));

// Types of activations and of cache codes.
constexpr int kBF16 = 0, kF16 = 1, kF32 = 2;
constexpr int kE4M3 = 0, kI8 = 1;

constexpr int elem_size(int t) { return t == kF32 ? 4 : 2; }

template <int T>
__device__ inline float elem_f32(const char* p) {
    if constexpr (T == kF32) return *reinterpret_cast<const float*>(p);
    else if constexpr (T == kF16) return static_cast<float>(*reinterpret_cast<const _Float16*>(p));
    else return __uint_as_float(static_cast<pg_u32>(*reinterpret_cast<const pg_u16*>(p)) << 16);
}
template <int T>
__device__ inline void store_elem(char* p, float x) {
    if constexpr (T == kF32) *reinterpret_cast<float*>(p) = x;
    else if constexpr (T == kF16) *reinterpret_cast<_Float16*>(p) = static_cast<_Float16>(x);
    else *reinterpret_cast<__bf16*>(p) = static_cast<__bf16>(x);
}

// Sum over the workgroup's threads of `v`, and the sum of those before this
// one.  One barrier pair; `lds` holds a value per wave.
template <int THREADS>
__device__ inline pg_i64 block_scan(pg_i64 v, pg_i64& total, pg_i64* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    pg_i64 x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const pg_i64 y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    pg_i64 before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        const pg_i64 y = lds[w];
        if (w < wave) before += y;
        sum += y;
    }
    __syncthreads();
    total = sum;
    return before + x - v;
}

// ---------------------------------------------------------------------------
// paged_plan
//
// Per request: old and new page counts ceil(length / page), ceil((length +
// count) / page); exclusive sums over the requests of the counts (its first
// row) and of the pages that it lacks (its first entry of the free list).  Per
// row: its request by binary search of the first rows, its page from the table
// or the free list, its slot.  The row at a page's first offset also writes
// that page's table entry: a page that is new to a request holds nothing older
// than its new tokens.  Bound by latency: a few KB move.  64 requests of a row
// each take 5 us in one launch, 4096 requests and 524288 rows (2 MB) 11 and 10 us
// in two.
// ---------------------------------------------------------------------------

struct PlanRequest {
    int start, length, first;  // first row, cached tokens, first entry of the free list
};

__device__ inline int page_count(pg_u32 tokens, pg_u32 page) { return static_cast<int>((tokens + (page - 1)) / page); }

// The sums, for all requests, in one workgroup; put(b, request, count)
// receives them.  Returns whether the plan fits; nothing has been put where it
// does not.  A request's length and count are read by one thread only, before
// it writes, so that new_lengths may be lengths.
template <int THREADS, class Put>
__device__ inline bool plan_requests(const PlanArgs& A, int& total_rows, Put put) {
    __shared__ pg_i64 lds[THREADS / 64];
    const pg_i64 per = (A.batch + THREADS - 1) / THREADS, b0 = threadIdx.x * per;
    const pg_i64 b1 = b0 + per < A.batch ? b0 + per : A.batch;
    const int used = *A.used, page = A.page;
    bool bad = used < 0;
    pg_i64 rows = 0, pages = 0;
    int length = 0, count = 0;
    for (pg_i64 b = b0; b < b1; ++b) {
        length = A.lengths[b * A.s_lengths];
        count = A.counts[b * A.s_counts];
        const pg_i64 all = static_cast<pg_i64>(length) + count;
        const bool wrong = length < 0 || count < 0 || all > 0x7FFFFFFF || all > A.width * page;
        bad |= wrong;
        if (wrong) continue;
        rows += count;
        pages += page_count(length + count, page) - page_count(length, page);
    }
    pg_i64 all_rows, all_pages;
    const pg_i64 row0 = block_scan<THREADS>(rows, all_rows, lds);
    const pg_i64 page0 = block_scan<THREADS>(pages, all_pages, lds);
    bad |= all_rows > A.rows || used + all_pages > A.nfree;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) *A.err = 4;
        return false;
    }
    total_rows = static_cast<int>(all_rows);
    int row = static_cast<int>(row0), first = used + static_cast<int>(page0);
    for (pg_i64 b = b0; b < b1; ++b) {
        if (per > 1) {
            length = A.lengths[b * A.s_lengths];
            count = A.counts[b * A.s_counts];
        }
        put(b, PlanRequest{row, length, first}, count);
        A.starts[b * A.s_starts] = row;
        A.new_lengths[b * A.s_new_lengths] = length + count;
        row += count;
        first += page_count(length + count, page) - page_count(length, page);
    }
    if (threadIdx.x == 0) {
        A.starts[A.batch * A.s_starts] = total_rows;
        *A.new_used = used + static_cast<int>(all_pages);
    }
    return true;
}

// Row r of request b.
__device__ inline void plan_row(const PlanArgs& A, int r, int b, PlanRequest q) {
    const int pos = q.length + (r - q.start), page = A.page;
    const int p = static_cast<int>(static_cast<pg_u32>(pos) / static_cast<pg_u32>(page)), off = pos - p * page;
    const int old = page_count(q.length, page);
    int id;
    if (p >= old) {
        id = A.free_pages[static_cast<pg_i64>(q.first + (p - old)) * A.s_free];
        if (off == 0) A.table[b * A.s_table + p * A.s_table_col] = id;
    } else {
        id = A.table[b * A.s_table + p * A.s_table_col];
    }
    const pg_i64 slot = static_cast<pg_i64>(id) * page + off;
    const bool fits = id >= 0 && slot <= 0x7FFFFFFF;
    if (!fits) *A.err = 5;
    A.slots[r * A.s_slots] = fits ? static_cast<int>(slot) : -1;
}

// One workgroup for everything: the requests' sums stay in LDS.
template <int THREADS, int BATCH>
__device__ inline void plan_one(const PlanArgs& A) {
    __shared__ int start[BATCH], length[BATCH], first[BATCH];
    int rows;
    const bool fits = plan_requests<THREADS>(A, rows, [&](pg_i64 b, PlanRequest q, int) {
        start[b] = q.start;
        length[b] = q.length;
        first[b] = q.first;
    });
    if (!fits) return;
    __syncthreads();
    const int n = static_cast<int>(A.batch);
    for (pg_i64 r = threadIdx.x; r < A.rows; r += THREADS) {
        if (r >= rows) {
            A.slots[r * A.s_slots] = -1;
            continue;
        }
        int lo = 0, hi = n;  // start[lo] <= r < start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= r) lo = mid;
            else hi = mid;
        }
        plan_row(A, static_cast<int>(r), lo, PlanRequest{start[lo], length[lo], first[lo]});
    }
}

// Two launches: the sums by one workgroup into the scratch, then the rows by
// as many workgroups as they need.
template <int THREADS>
__device__ inline void plan_sums(const PlanArgs& A) {
    int* const start = A.scratch + 2;
    int* const length = start + A.batch;
    int* const first = length + A.batch;
    int rows;
    const bool fits = plan_requests<THREADS>(A, rows, [&](pg_i64 b, PlanRequest q, int) {
        start[b] = q.start;
        length[b] = q.length;
        first[b] = q.first;
    });
    if (threadIdx.x == 0) {
        A.scratch[0] = fits;
        A.scratch[1] = fits ? rows : 0;
    }
}

template <int THREADS>
__device__ inline void plan_rows(const PlanArgs& A) {
    if (!A.scratch[0]) return;
    const int rows = A.scratch[1];
    const int* const start = A.scratch + 2;
    const int* const length = start + A.batch;
    const int* const first = length + A.batch;
    const pg_i64 r0 = static_cast<pg_i64>(blockIdx.x) * kPlanRows;
    const pg_i64 end = r0 + kPlanRows < A.rows ? r0 + kPlanRows : A.rows;
    const int r1 = static_cast<int>(end < rows ? end : rows);  // rows with a token
    if (r0 < r1) {
        // The requests of the first and the last row: the whole workgroup probes.
        int lo[2] = {0, 0}, hi[2] = {static_cast<int>(A.batch), static_cast<int>(A.batch)};
        const int row[2] = {static_cast<int>(r0), r1 - 1};
        while (hi[0] - lo[0] > 1 || hi[1] - lo[1] > 1) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int step = (hi[k] - lo[k] + THREADS - 1) / THREADS;
                const int at = lo[k] + static_cast<int>(threadIdx.x) * step;
                const int below = __syncthreads_count(at < hi[k] && start[at] <= row[k]);
                lo[k] += (below - 1) * step;
                hi[k] = lo[k] + step < hi[k] ? lo[k] + step : hi[k];
            }
        }
        for (int r = static_cast<int>(r0) + static_cast<int>(threadIdx.x); r < r1; r += THREADS) {
            int l = lo[0], h = hi[1];
            while (h - l > 1) {
                const int mid = (l + h) >> 1;
                if (start[mid] <= r) l = mid;
                else h = mid;
            }
            plan_row(A, r, l, PlanRequest{start[l], length[l], first[l]});
        }
    }
    for (pg_i64 r = (r0 > rows ? r0 : rows) + threadIdx.x; r < end; r += THREADS) A.slots[r * A.s_slots] = -1;
}

// ---------------------------------------------------------------------------
// Codes
// ---------------------------------------------------------------------------

template <int CT>
constexpr float code_top() {
    return CT == kI8 ? 127.0f : 448.0f;
}

// Two codes (bytes 0, 1 or 2, 3 of w) as two bf16 or f16 values: exact, both
// types hold the 4 significant bits of e4m3 and the 8 of a signed byte.
template <int CT, bool H, bool HI>
__device__ inline pg_u32 codes2(pg_u32 w) {
    if constexpr (CT == kE4M3) {
        if constexpr (H) return __builtin_bit_cast(pg_u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
        else return __builtin_bit_cast(pg_u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    } else {
        if constexpr (H) {
            // The f16 of bits 0x6400 + u is 1024 + u; u is the code + 128.
            const pg_u32 x = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, HI ? 0x04030402u : 0x04010400u);
            return __builtin_bit_cast(pg_u32, __builtin_bit_cast(pg_h2, x) - pg_h2{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)});
        }
        const float a = static_cast<float>(static_cast<signed char>(w >> (HI ? 16 : 0)));
        const float b = static_cast<float>(static_cast<signed char>(w >> (HI ? 24 : 8)));
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
}

// Four numbers, already multiplied by 1 / scale, as codes.  INSIDE: none is NaN,
// and none beyond the largest code by more than a few roundings of float32,
// which round away again.
template <int CT, bool INSIDE>
__device__ inline pg_u32 encode4(const float* y) {
    constexpr float top = code_top<CT>();
    float z[4];
    bool nan[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        nan[i] = !INSIDE && y[i] != y[i];
        z[i] = INSIDE ? y[i] : fminf(fmaxf(y[i], -top), top);
    }
    pg_u32 w;
    if constexpr (CT == kI8) {
        // 1.5 * 2^23 more: rounded to a whole number whose byte is the lowest.
        pg_u32 c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = __float_as_uint((nan[i] ? 0.0f : z[i]) + 0x1.8p23f);
        w = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u), __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u), 0x05040100u);
    } else {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], c, true);
        w = static_cast<pg_u32>(c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (nan[i]) w = (w & ~(0xFFu << (8 * i))) | 0x7Fu << (8 * i);
    }
    return w;
}

template <int CT>
__device__ inline float decode1(pg_u32 w, int i) {
    const pg_u32 byte = (w >> (8 * i)) & 0xFFu;
    if constexpr (CT == kI8) return static_cast<float>(static_cast<signed char>(byte));
    else return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(byte), 0);
}

// ---------------------------------------------------------------------------
// paged_store
//
// One wave per run of neighbouring rows of a page, head, and keys or values:
// the largest finite |x| of the run, the scale (kept tokens: at least the old
// one), the kept codes anew where it grew, the run's codes.  Every quotient is
// the product with 1 / scale, rounded as float32 values are, so that the codes
// follow from the inputs bit by bit.  Infinities and NaN are met only where the
// run's largest bits say so; their runs are read a second time.  16000 rows of
// 2 x 8 heads of 128 in bf16 to e4m3 (101 MB): 23 us, 4.4 TB/s; with NaN tests and
// clamps on every element and 64-bit indices 37, bound by instructions.
// ---------------------------------------------------------------------------

typedef unsigned short pg_us2 __attribute__((ext_vector_type(2)));
template <bool V>
struct Flag {
    static constexpr bool value = V;
};

// Eight elements of x at p, as they are.
template <int T>
struct Eight {
    pg_u32 w[T == kF32 ? 8 : 4];
};
template <int T, bool VEC>
__device__ inline void load8(const char* p, Eight<T>& x) {
    constexpr int N = T == kF32 ? 8 : 4;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if constexpr (VEC) {
            const pg_u32x4 a = *reinterpret_cast<const pg_u32x4*>(p + 4 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) x.w[i + k] = a[k];
        } else {
#pragma unroll
            for (int k = i; k < i + 4; ++k) {
                if constexpr (T == kF32) {
                    x.w[k] = *reinterpret_cast<const pg_u32*>(p + 4 * k);
                } else {
                    x.w[k] = static_cast<pg_u32>(*reinterpret_cast<const pg_u16*>(p + 4 * k)) |
                             static_cast<pg_u32>(*reinterpret_cast<const pg_u16*>(p + 4 * k + 2)) << 16;
                }
            }
        }
    }
}
template <int T>
__device__ inline void values8(const Eight<T>& x, float* y) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (T == kF32) {
            y[i] = __uint_as_float(x.w[i]);
        } else if constexpr (T == kF16) {
            const pg_u32 w = x.w[i >> 1];
            y[i] = static_cast<float>(__builtin_bit_cast(pg_h2, w)[i & 1]);
        } else {
            y[i] = __uint_as_float(i & 1 ? x.w[i >> 1] & 0xFFFF0000u : x.w[i >> 1] << 16);
        }
    }
}
// The largest |x| as bits without sign, which are ordered as the numbers are,
// NaN above infinity; of 16-bit types two at once.
template <int T>
__device__ inline pg_u32 most8(const Eight<T>& x, pg_u32 most) {
#pragma unroll
    for (int i = 0; i < (T == kF32 ? 8 : 4); ++i) {
        if constexpr (T == kF32) {
            const pg_u32 a = x.w[i] & 0x7FFFFFFFu;
            most = a > most ? a : most;
        } else {
            const pg_u32 a = x.w[i] & 0x7FFF7FFFu;
            most = __builtin_bit_cast(pg_u32, __builtin_elementwise_max(__builtin_bit_cast(pg_us2, a), __builtin_bit_cast(pg_us2, most)));
        }
    }
    return most;
}

template <int D, int PAGE, int T, int CT, bool VEC, int CHUNK>
__device__ inline void store_rows(const StoreArgs& A) {
    const int heads = A.heads;
    constexpr int PARTS = D / 8;  // pieces of eight elements in a row
    // Pieces that a lane holds: a page's, of 64 registers at most.
    constexpr int NEED = (PAGE * PARTS + 63) / 64, ROUNDS = NEED < 8 ? NEED : 8;
    const int lane = threadIdx.x & 63;
    // Fewer than 2^24 workgroups of four waves.
    const pg_u32 item = blockIdx.x * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const pg_u32 chunk = item / static_cast<pg_u32>(2 * heads);
    const int which = static_cast<int>(item - chunk * static_cast<pg_u32>(2 * heads)), h = which >> 1, kv = which & 1;
    const pg_i64 row0 = static_cast<pg_i64>(chunk) * CHUNK;
    if (row0 >= A.rows) return;
    const pg_i64 slots_end = A.pages * PAGE;
    auto page_of = [&](pg_i64 r) -> int {  // -1: not stored
        if (r < 0 || r >= A.rows) return -1;
        const int s = A.slots[r * A.s_slots];
        return s < 0 || s >= slots_end ? -1 : s / PAGE;
    };
    // The runs that begin among the chunk's rows.
    pg_u64 leaders;
    {
        const pg_i64 r = row0 + lane;
        const int p = lane < CHUNK ? page_of(r) : -1;
        if (lane < CHUNK && r < A.rows && A.slots[r * A.s_slots] >= slots_end) *A.err = 6;
        leaders = __ballot(p >= 0 && page_of(r - 1) != p);
    }
    const char* const x = A.x[kv] + h * A.s_x[kv][1] * elem_size(T);
    while (leaders) {
        const pg_i64 r0 = row0 + __builtin_ctzll(leaders);
        leaders &= leaders - 1;
        const int page = page_of(r0);
        // Rows of the run, its first offset, and whether its offsets ascend by one.
        int n = 0, low = PAGE;
        bool dense = true;
        for (;;) {
            const bool in = page_of(r0 + n + lane) == page;
            const pg_u64 out = ~__ballot(in);
            const int more = out ? __builtin_ctzll(out) : 64;
            const int off = lane < more ? A.slots[(r0 + n + lane) * A.s_slots] - page * PAGE : PAGE;
            if (n == 0) low = __builtin_amdgcn_readfirstlane(off);
            dense = dense && __ballot(lane < more && off != low + n + lane) == 0;
            if (!dense) {
                int l = off;
#pragma unroll
                for (int d = 32; d >= 1; d >>= 1) {
                    const int y = __shfl_xor(l, d, 64);
                    l = y < l ? y : l;
                }
                low = l < low ? l : low;
            }
            n += more;
            if (more < 64) break;
        }
        const char* const xr = x + r0 * A.s_x[kv][0] * elem_size(T);
        auto from = [&](int t, int part) { return xr + (t * A.s_x[kv][0] + part * 8) * elem_size(T); };
        // The run's first pieces stay in registers, all their loads in flight at
        // once; what is longer (or not in order) is read a second time.
        Eight<T> held[ROUNDS];
        const char* const own = from(lane / PARTS, lane % PARTS);
        pg_u32 bits = 0;
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k) {
            const int e = lane + 64 * k;
            held[k] = {};
            if (e < n * PARTS) load8<T, VEC>(64 % PARTS == 0 ? own + k * (64 / PARTS) * A.s_x[kv][0] * elem_size(T) : from(e / PARTS, e % PARTS), held[k]);
        }
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k) bits = most8<T>(held[k], bits);
        for (int e = lane + 64 * ROUNDS; e < n * PARTS; e += 64) {
            Eight<T> x8;
            load8<T, VEC>(from(e / PARTS, e % PARTS), x8);
            bits = most8<T>(x8, bits);
        }
        if constexpr (T != kF32) bits = (bits & 0xFFFFu) > bits >> 16 ? bits & 0xFFFFu : bits >> 16;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            const pg_u32 y = static_cast<pg_u32>(__shfl_xor(static_cast<int>(bits), d, 64));
            bits = y > bits ? y : bits;
        }
        constexpr pg_u32 kInf = T == kF32 ? 0x7F800000u : T == kF16 ? 0x7C00u : 0x7F80u;
        const bool finite = __builtin_amdgcn_readfirstlane(bits) < kInf;
        float most = 0.0f;
        if (finite) {
            Eight<T> x8 = {};
            float y[8];
            x8.w[0] = bits;
            values8<T>(x8, y);
            most = y[0];
        } else {
            for (int e = lane; e < n * PARTS; e += 64) {
                Eight<T> x8;
                float y[8];
                load8<T, VEC>(from(e / PARTS, e % PARTS), x8);
                values8<T>(x8, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = fabsf(y[i]);
                    if (a < __builtin_inff()) most = fmaxf(most, a);
                }
            }
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
        }
        float* const sp = A.scale[kv] + page * A.s_scale[kv][0] + h * A.s_scale[kv][1];
        const float old = low > 0 ? *sp : 0.0f;
        const float scale = fmaxf(fmaxf(most / code_top<CT>(), 0x1p-126f), old);
        const float inverse = 1.0f / scale;
        char* const cp = A.cache[kv] + page * A.s_cache[kv][0] + h * A.s_cache[kv][1];
        if (low > 0 && scale > old) {
            for (int e = lane; e < low * PARTS; e += 64) {
                const int t = e / PARTS;
                pg_u32x2* const c = reinterpret_cast<pg_u32x2*>(cp + t * A.s_cache[kv][2] + (e - t * PARTS) * 8);
                pg_u32x2 w = *c;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = (decode1<CT>(w[k], i) * old) * inverse;
                    w[k] = encode4<CT, false>(y);
                }
                *c = w;
            }
        }
        auto code = [&](auto inside, const Eight<T>& x8, char* to) {
            constexpr bool INSIDE = decltype(inside)::value;
            float y[8];
            values8<T>(x8, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = y[i] * inverse;
            *reinterpret_cast<pg_u32x2*>(to) = pg_u32x2{encode4<CT, INSIDE>(y), encode4<CT, INSIDE>(y + 4)};
        };
        auto put = [&](int t, int part, int off) {
            Eight<T> x8;
            load8<T, VEC>(from(t, part), x8);
            code(Flag<false>(), x8, cp + off * A.s_cache[kv][2] + part * 8);
        };
        if (dense && finite) {
            char* const to = cp + (low + lane / PARTS) * A.s_cache[kv][2] + lane % PARTS * 8;
#pragma unroll
            for (int k = 0; k < ROUNDS; ++k) {
                const int e = lane + 64 * k;
                if (e < n * PARTS)
                    code(Flag<true>(), held[k],
                         64 % PARTS == 0 ? to + k * (64 / PARTS) * A.s_cache[kv][2] : cp + (low + e / PARTS) * A.s_cache[kv][2] + e % PARTS * 8);
            }
            for (int e = lane + 64 * ROUNDS; e < n * PARTS; e += 64) put(e / PARTS, e % PARTS, low + e / PARTS);
        } else {
            // Rows in order, each piece by the same lane: of several rows at one
            // offset the last one stays.
            for (int t = 0; t < n; ++t)
                for (int part = lane; part < PARTS; part += 64) put(t, part, A.slots[(r0 + t) * A.s_slots] - page * PAGE);
        }
        if (lane == 0) *sp = scale;
    }
}

// ---------------------------------------------------------------------------
// paged_attention
//
// A unit is C tokens of one request times the G query heads of one key head:
// up to RB = 16 * NT query rows that read the same keys.  A workgroup's four
// waves take 32 of every 128 tokens each, with a softmax of their own, and are
// joined through LDS.  All tiles of all units make one line that the
// workgroups cut into equal pieces, so a long request is shared by many of
// them; the pieces of a unit that is cut meet in join().
//
// Per 32 tokens a wave forms S^T = K q^T and O^T += V^T P^T with
// v_mfma_f32_16x16x32: both operands' lanes hold what their loads deliver.
//   K: lane (m, g) of 16 x 4 reads 16 bytes of token m, dims 64j + 16g, which
//      are two MFMA operands; q is laid out alike.
//   S: lane (n, g) holds, of query row n, tokens 4g .. 4g + 3 of each 16: the
//      eight of a lane are the P operand of one MFMA, in that order of tokens.
//   V: lane (c, g) reads those eight tokens' dims 64j + 4c .. + 3, one dword
//      each; byte q of them is the operand of dims 64j + 4c + q.
//   O: lane (n, g) ends up with dims 64j + 16g .. + 15 of query row n.
// No value crosses lanes but the maxima, and those only when one grows: p is
// exp2(s - m) for an m that may lag the true maximum by a factor of 2^8.
// Codes enter the MFMAs as they are, exactly; a page's scales multiply s and p
// in float32.  q enters exactly too (an f32 as three bf16), p as two bf16
// parts (2^-16 of it; three for f32 outputs), sums are float32.
//
// 64 requests of 512 to 8192 tokens, 8 x 4 heads of 128 (606 MB of e4m3): 116 us,
// 5.2 TB/s, from 2 KB pieces of pages; both launches 122 us, and 84 us with all
// requests on the same 64 pages, which L2 holds: bytes and instructions take about
// as long, and overlap in part only.  Two requests of about 100000 tokens, f16
// over int8 (479 MB): 94 us, 5.1 TB/s.
// ---------------------------------------------------------------------------

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline pg_i64 uniform64(pg_i64 x) {
    const pg_u32 lo = __builtin_amdgcn_readfirstlane(static_cast<int>(x));
    const pg_u32 hi = __builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32));
    return static_cast<pg_i64>(static_cast<pg_u64>(hi) << 32 | lo);
}

template <int D_, int PAGE_, int G_, int NT_, int QT_, int CT_, bool WIN_, bool LSE_, bool VEC_, bool PROMPT_ = false>
struct Attend {
    static constexpr bool PROMPT = PROMPT_;
    static constexpr int D = D_, PAGE = PAGE_, G = G_, NT = NT_, QT = QT_, CT = CT_;
    static constexpr bool WIN = WIN_, LSE = LSE_, VEC = VEC_;
    static constexpr int RB = 16 * NT;
    static constexpr int C = G <= RB ? RB / G : 1;               // tokens of a unit
    static constexpr int HS = G <= RB ? 1 : (G + RB - 1) / RB;   // units that share a token's heads
    static constexpr int GH = G <= RB ? G : RB;                  // query heads of a unit
    static constexpr int NK = (D + 63) / 64, DP = 64 * NK;
    static constexpr bool H = QT == kF16;                        // K and q as f16
    static constexpr int QP = QT == kF32 ? 3 : 1;                // parts of q
    static constexpr int PP = QT == kF32 ? 3 : 2;                // parts of p
    static constexpr bool PAGED16 = PAGE % 16 == 0;              // 16 aligned tokens lie in one page
    static constexpr int PART = RB * (2 + DP);                   // floats of a partial result
    static constexpr int E = 16 * NK * NT;                       // accumulators of a lane

    // One request.
    struct Request {
        int row, n, length, first, kt, units;  // first row, rows, tokens; first tile, tiles and units of a key head
        bool bad;
    };
    __device__ static Request request(const AttendArgs& A, pg_i64 b, bool report) {
        Request r;
        const int s0 = A.starts[b * A.s_starts], s1 = A.starts[(b + 1) * A.s_starts];
        int length = A.lengths[b * A.s_lengths];
        const pg_i64 most = A.width * PAGE;
        const bool bad = s0 < 0 || s1 < s0 || s1 > A.rows || length < 0 || length > most;
        if (bad && report) *A.err = 7;
        r.bad = bad;
        if (bad || (PROMPT ? s1 - s0 <= A.few : s1 - s0 > A.few)) {
            r.row = r.n = r.length = r.first = r.kt = r.units = 0;
            return r;
        }
        r.row = s0;
        r.n = s1 - s0;
        r.length = length;
        int lo = 0;
        if constexpr (WIN) {
            const pg_i64 w = static_cast<pg_i64>(length) - r.n + 1 - A.window;
            lo = w > 0 ? static_cast<int>(w) : 0;
            if (lo > length) lo = length;
        }
        r.first = lo / kAttendTile;
        const int last = static_cast<int>((static_cast<pg_u32>(length) + (kAttendTile - 1)) / kAttendTile);
        r.kt = last > r.first ? last - r.first : 1;
        r.units = (r.n + C - 1) / C * HS;
        return r;
    }

    static constexpr int SC = PAGED16 ? 2 : 1;
    struct Raw {
        pg_u32x4 k[2][NK];
        pg_u32 v[NK][8];
        float ks[SC], vs[SC];  // scales: of each 16 tokens; over odd pages of token base + lane % 32
    };
    // This lane's number, for what is computed from it where it is used: the
    // compiler would compute that ahead of the loops over tokens and carry it
    // through them, beyond the registers that there are.
    __device__ static int own_lane() {
        pg_u32 all = ~0u;
        asm volatile("" : "+s"(all));
        return static_cast<int>(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0)));
    }
    // x of lane `first` + `more`: 4 * first in a register, the constant in the instruction.
    __device__ static int of_lane(int first4, int more, int x) { return __builtin_amdgcn_ds_bpermute(first4 + 4 * more, x); }
    // The four lanes n + 16 g of a query row joined, in each of them.
    template <class Op>
    __device__ static float over_groups(float x, Op op) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
        const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
    }
    // The scales of the tokens in this lane's places.
    __device__ static void scales_of(const float (&s)[SC], float (&f)[8]) {
        const int first4 = PAGED16 ? 0 : own_lane() & 48;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = PAGED16 ? s[e >> 2] : __int_as_float(of_lane(first4, 4 * (e & 4) + (e & 3), __float_as_int(s[0])));
    }

    // One unit of one workgroup's piece.
    struct Unit {
        const int* table;  // the request's row
        int h, n;          // key head; tokens of the unit
        int p0;            // position of its first token
        int lo, hi;        // positions that its rows attend to, together
        const char* cache[2];  // the key head's first page, keys and values, and their scales
        const float* scale[2];
        __device__ void aim(const AttendArgs& A, int head) {
            h = head;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                cache[i] = A.cache[i] + h * A.s_cache[i][1];
                scale[i] = A.scale[i] + h * A.s_scale[i][1];
            }
        }
    };
    // Elements before page `id`: the host has checked that a page's stride has 32 bits.
    __device__ static pg_i64 pages_on(int id, long long stride) {
        return static_cast<pg_i64>(static_cast<pg_u64>(static_cast<pg_u32>(id)) * static_cast<pg_u32>(stride));
    }
    // Elements before token `off` of a page, up to 4095 strides of 2^26; 16 of them
    // have 32 bits.  Neither is negative: as a signed product it takes more scalar
    // registers, which the tile kernel beside it then lacks (8192-token prompts of
    // head size 64: 120 us, so 112).
    __device__ static pg_i64 token_at(int off, long long stride) { return pages_on(off, stride); }

    // Pages of the 32 tokens from `base` on.  Tokens outside the unit's
    // positions take the page of a neighbour inside; they are masked.
    static constexpr int IDS = PAGE % 32 == 0 ? 1 : 2;
    struct Pages {
        int id[IDS];
    };
    __device__ static int checked(const AttendArgs& A, int id) {
        const bool out = static_cast<pg_u32>(id) >= static_cast<pg_u32>(A.pages);
        if (__ballot(out)) *A.err = 7;
        return out ? 0 : id;
    }

    // First dims of a lane's piece j of a key (16 dims) and of a value (4).  Where
    // the head size ends inside 64 dims, pieces behind it repeat the row's last
    // one: q is 0 there, a NaN is in the scores either way, and those dims of the
    // output are not written.  So no load stands under a branch that only some
    // lanes take.  The compiler may put copies and spills of other values at the
    // end of such a branch before it gives the other lanes their turn, which then
    // go on with what the register or the spill slot held before: 7 rows over int8
    // pages of 8 tokens, head size 80, lost rows 4 to 6 that way, on some runs.
    __device__ static int key_dim(int j, int g) {
        const int d = 64 * j + 16 * g;
        return D % 64 != 0 && j == NK - 1 && d > D - 16 ? D - 16 : d;
    }
    __device__ static int value_dim(int j, int m) {
        const int d = 64 * j + 4 * m;
        return D % 64 != 0 && j == NK - 1 && d > D - 4 ? D - 4 : d;
    }
    __device__ static int inside(const Unit& u, int t) { return t < u.lo ? u.lo : t >= u.hi ? u.hi - 1 : t; }
    __device__ static void pages(const AttendArgs& A, const Unit& u, int base, Pages& p) {
        if constexpr (PAGED16) {
#pragma unroll
            for (int i = 0; i < IDS; ++i) p.id[i] = shared_load(u.table + inside(u, base + 16 * i) / PAGE);
        } else {
            p.id[0] = u.table[inside(u, base + (static_cast<int>(threadIdx.x) & 31)) / PAGE];
        }
    }

    __device__ static void load(const AttendArgs& A, const Unit& u, int base, const Pages& p, Raw& r) {
        const int lane = D % 64 != 0 ? own_lane() : threadIdx.x & 63, m = lane & 15, g = lane >> 4;
        if constexpr (PAGED16) {
            const char* page[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int off = (base + 16 * i) % PAGE;
                if (i < IDS) {
                    const int id = checked(A, uniform(p.id[i]));
                    r.ks[i] = shared_load(u.scale[0] + pages_on(id, A.s_scale[0][0]));
                    r.vs[i] = shared_load(u.scale[1] + pages_on(id, A.s_scale[1][0]));
                    page[0] = u.cache[0] + pages_on(id, A.s_cache[0][0]);
                    page[1] = u.cache[1] + pages_on(id, A.s_cache[1][0]);
                } else {
                    r.ks[i] = r.ks[0];
                    r.vs[i] = r.vs[0];
                }
                const char* const kp = page[0] + token_at(off, A.s_cache[0][2]);
                const char* const vp = page[1] + token_at(off, A.s_cache[1][2]);
                const int ko = m * static_cast<int>(A.s_cache[0][2]), vt = static_cast<int>(A.s_cache[1][2]);
#pragma unroll
                for (int j = 0; j < NK; ++j) r.k[i][j] = *reinterpret_cast<const pg_u32x4*>(kp + ko + key_dim(j, g));
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int t = 0; t < 4; ++t) r.v[j][4 * i + t] = *reinterpret_cast<const pg_u32*>(vp + (4 * g + t) * vt + value_dim(j, m));
            }
        } else {
            // Lane l has looked up token base + l % 32.
            const int id = checked(A, p.id[0]), off = inside(u, base + (lane & 31)) % PAGE;
            const int own = own_lane(), m4 = 4 * (own & 15), g4 = own & 48;
            r.ks[0] = u.scale[0][pages_on(id, A.s_scale[0][0])];
            r.vs[0] = u.scale[1][pages_on(id, A.s_scale[1][0])];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const char* const row = u.cache[0] + pages_on(of_lane(m4, 16 * i, id), A.s_cache[0][0]) + token_at(of_lane(m4, 16 * i, off), A.s_cache[0][2]);
#pragma unroll
                for (int j = 0; j < NK; ++j) r.k[i][j] = *reinterpret_cast<const pg_u32x4*>(row + key_dim(j, g));
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int more = (t & 4) * 4 + (t & 3);
                const char* const row = u.cache[1] + pages_on(of_lane(g4, more, id), A.s_cache[1][0]) + token_at(of_lane(g4, more, off), A.s_cache[1][2]);
#pragma unroll
                for (int j = 0; j < NK; ++j) r.v[j][t] = *reinterpret_cast<const pg_u32*>(row + value_dim(j, m));
            }
        }
    }

    __device__ static pg_f32x4 mma(pg_u32x4 a, pg_u32x4 b, pg_f32x4 c, bool half) {
        if (half) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_h8, a), __builtin_bit_cast(pg_h8, b), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf8, a), __builtin_bit_cast(pg_bf8, b), c, 0, 0, 0);
    }
    // Two floats as bf16, and what the rounding left of them.
    __device__ static pg_u32 take_bf16(float& a, float& b) {
        const pg_bf2 h = __builtin_convertvector((pg_f32x2{a, b}), pg_bf2);
        const pg_u32 w = __builtin_bit_cast(pg_u32, h);
        a = a - __uint_as_float(w << 16);
        b = b - __uint_as_float(w & 0xFFFF0000u);
        return w;
    }

    struct State {
        pg_u32x4 q[NT][2 * NK][QP];
        pg_f32x4 o[NT][NK][4];
        float m[NT], l[NT];
    };

    __device__ static void load_q(const AttendArgs& A, const Unit& u, int row, int head, State& st) {
        const int lane = own_lane(), n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            // Places without a row or a dim read the unit's first row, or a dim inside, and are 0.
            const int r = 16 * t + n, i = r / GH, hh = r - i * GH;
            const bool valid = i < u.n && (HS == 1 || head % G + hh < G);
            const char* const p = A.q + ((row + (valid ? i : 0)) * A.s_q[0] + (head + (valid ? hh : 0)) * A.s_q[1]) * elem_size(QT);
#pragma unroll
            for (int j = 0; j < 2 * NK; ++j) {
                const int d = 64 * (j >> 1) + 16 * g + 8 * (j & 1);
                const bool in = valid && (D % 64 == 0 || d < D);
                Eight<QT> x8;
                load8<QT, VEC>(p + (D % 64 != 0 && d >= D ? D - 8 : d) * elem_size(QT), x8);
                if constexpr (QT == kF32) {
                    float x[8];
                    values8<QT>(x8, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = in ? x[e] : 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int k = 0; k < 3; ++k) st.q[t][j][k][e] = take_bf16(x[2 * e], x[2 * e + 1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.q[t][j][0][e] = in ? x8.w[e] : 0;
                }
            }
            st.m[t] = -__builtin_inff();
            st.l[t] = 0.0f;
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[t][j][e] = pg_f32x4{0, 0, 0, 0};
        }
    }

    // Four codes, kept in one register: the compiler would carry their bytes from
    // the loads through the loop in one each.
    __device__ static pg_u32 whole(pg_u32 w) {
        asm("" : "+v"(w));
        return w;
    }

    // O^T += V^T P^T for P's parts in the eight token places of a lane.
    __device__ static void values(const pg_u32 (&v)[NK][8], const pg_u32x4 (&p)[NT][PP], pg_f32x4 (&o)[NT][NK][4]) {
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            pg_u32x4 a[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const pg_u32 x = whole(v[j][2 * e]), y = whole(v[j][2 * e + 1]);
                const pg_u32 w0 = __builtin_amdgcn_perm(y, x, 0x05010400u), w1 = __builtin_amdgcn_perm(y, x, 0x07030602u);
                a[0][e] = codes2<CT, false, false>(w0);
                a[1][e] = codes2<CT, false, true>(w0);
                a[2][e] = codes2<CT, false, false>(w1);
                a[3][e] = codes2<CT, false, true>(w1);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < PP; ++k) o[t][j][q] = mma(a[q], p[t][k], o[t][j][q], false);
        }
    }

    // p of the scores, and its products with the values.
    __device__ static void weigh(const Raw& r, const float (&s)[NT][8], State& st) {
        pg_u32x4 p[NT][PP];
        float vs[8];
        scales_of(r.vs, vs);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float m = st.m[t] == -__builtin_inff() ? 0.0f : st.m[t];
            float x[8], l = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(s[t][e] - m);
                l += x[e];
                x[e] *= vs[e];
            }
            st.l[t] += l;
#pragma unroll
            for (int k = 0; k < PP; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[t][k][e] = take_bf16(x[2 * e], x[2 * e + 1]);
        }
        values(r.v, p, st.o);
    }

    // For a branch that is hardly ever taken: what it computes of these is not
    // moved ahead of it, where it would take registers from every step.
    __device__ static void apart(Raw& r, float (&s)[NT][8]) {
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(r.v[j][e]));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(s[t][e]));
    }

    // Scores and values of a step that some row does not see whole.  What lies
    // outside the unit's positions may be anything; a NaN among values that some
    // rows see and others do not (0 * NaN is NaN) goes into those rows' sums here
    // and is 0 afterwards: ones at the NaNs times ones at the rows that see them.
    __device__ static void mask(const AttendArgs& A, const Unit& u, int base, Raw& r, float (&s)[NT][8], State& st) {
        const int lane = own_lane(), n = lane & 15, g = lane >> 4;
        const int tok = base + 4 * g;  // token of place e: tok + e % 4, 16 further for e >= 4
        pg_u32 seen[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int hi = u.p0 + (16 * t + n) / GH + 1, lo = WIN ? hi - A.window : 0;
            seen[t] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = tok + (e & 3) + 4 * (e & 4);
                const bool in = at < hi && at >= lo && at < u.hi;
                seen[t] |= static_cast<pg_u32>(in) << e;
                s[t][e] = in ? s[t][e] : -__builtin_inff();
            }
        }
        pg_u32 nan = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int at = tok + (e & 3) + 4 * (e & 4);
            const bool in = at < u.hi && at >= u.lo;
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                r.v[j][e] = in ? r.v[j][e] : 0;
                nan |= ((r.v[j][e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
            }
        }
        if constexpr (CT == kE4M3 && (C > 1 || WIN)) {
            if (__ballot(nan != 0) == 0) return;
            apart(r, s);
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                pg_u32 ones[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const pg_u32 at = (((r.v[j][e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
                    ones[e] = at * 0x38u;  // the code of 1
                    r.v[j][e] &= ~(at * 0xFFu);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    pg_u32x4 a;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const pg_u32 w = __builtin_amdgcn_perm(ones[2 * e + 1], ones[2 * e], q < 2 ? 0x05010400u : 0x07030602u);
                        a[e] = q & 1 ? codes2<CT, false, true>(w) : codes2<CT, false, false>(w);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        pg_u32x4 p;
                        pg_u32 at = seen[t];
                        asm volatile("" : "+v"(at));  // p is made where it is used
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[e] = (at >> (2 * e) & 1) * 0x3F80u | (at >> (2 * e + 1) & 1) * 0x3F800000u;
                        const pg_f32x4 hit = mma(a, p, pg_f32x4{0, 0, 0, 0}, false);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (hit[i] > 0.0f) st.o[t][j][q][i] = __builtin_nanf("");
                    }
                }
            }
        }
    }

    __device__ static void step(const AttendArgs& A, const Unit& u, int base, Raw& r, State& st) {
        float s[NT][8];
        {
            pg_f32x4 acc[NT][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t][i] = pg_f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 2 * NK; ++j) {
                    const pg_u32 w0 = whole(r.k[i][j >> 1][2 * (j & 1)]), w1 = whole(r.k[i][j >> 1][2 * (j & 1) + 1]);
                    const pg_u32x4 a = {codes2<CT, H, false>(w0), codes2<CT, H, true>(w0), codes2<CT, H, false>(w1), codes2<CT, H, true>(w1)};
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int k = 0; k < QP; ++k) acc[t][i] = mma(a, st.q[t][j][k], acc[t][i], H);
                }
            }
            float ks[8];
            scales_of(r.ks, ks);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = ks[e] * A.factor;
#pragma unroll
                for (int t = 0; t < NT; ++t) s[t][e] = acc[t][e >> 2][e & 3] * f;
            }
        }
        // Every row of the unit sees every one of the tokens, or not.
        if (!(base + 32 <= u.p0 + 1 && (!WIN || base >= u.p0 + u.n - A.window))) mask(A, u, base, r, s, st);
        // The maximum, only if some score is far above it.
        bool grow = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float mx = s[t][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[t][e]);
            grow |= mx > st.m[t] + 8.0f;
        }
        if (__ballot(grow)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float mx = s[t][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[t][e]);
                mx = over_groups(mx, [](float a, float b) { return fmaxf(a, b); });
                const float m = fmaxf(st.m[t], mx);
                const float a = m == st.m[t] ? 1.0f : __builtin_amdgcn_exp2f(st.m[t] - m);
                st.m[t] = m;
                st.l[t] *= a;
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) st.o[t][j][q] *= a;
            }
        }
        weigh(r, s, st);
    }

    __device__ static void write_row(const AttendArgs& A, int row, int head, int g, int j, const pg_f32x4 (&o)[4], float f) {
        // o[q][i]: dim 64j + 16g + 4i + q.
        const int d = 64 * j + 16 * g;
        if (D % 64 != 0 && d >= D) return;
        char* const p = A.out + (row * A.s_out[0] + head * A.s_out[1] + d) * elem_size(QT);
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = o[i & 3][i >> 2] * f;
        if constexpr (VEC && QT == kF32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<pg_f32x4*>(p + 16 * i) = pg_f32x4{y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]};
        } else if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                pg_u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = y[8 * i + 2 * e], b = y[8 * i + 2 * e + 1];
                    if constexpr (QT == kF16) w[e] = __builtin_bit_cast(pg_u32, (pg_h2{static_cast<_Float16>(a), static_cast<_Float16>(b)}));
                    else w[e] = __builtin_bit_cast(pg_u32, __builtin_convertvector((pg_f32x2{a, b}), pg_bf2));
                }
                *reinterpret_cast<pg_u32x4*>(p + 16 * i) = w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) store_elem<QT>(p + i * elem_size(QT), y[i]);
        }
    }

    struct Shared {
        pg_f32x4 o[4][NT * NK * 4][64];
        float m[4][RB], l[4][RB];
        pg_i64 scan[4];
        pg_i64 begin[2];  // where the piece starts: request, items before it
    };

    __device__ static void run(const AttendArgs& A, int workgroup, Shared& sh) {
        const int wave = uniform(threadIdx.x >> 6);
        const pg_i64 w = workgroup;
        int* const span = A.spans + w * kSpanInts;
        // The pieces: per request the items of its units, and their sums.
        const pg_i64 per = (A.batch + kAttendThreads - 1) / kAttendThreads, b0 = threadIdx.x * per;
        const pg_i64 b1 = b0 + per < A.batch ? b0 + per : A.batch;
        pg_i64 sum = 0;
        for (pg_i64 b = b0; b < b1; ++b) {
            const Request r = request(A, b, w == 0);
            sum += static_cast<pg_i64>(A.heads) * r.units * r.kt;
        }
        pg_i64 total;
        pg_i64 before = block_scan<kAttendThreads>(sum, total, sh.scan);
        total = uniform64(total);
        const pg_i64 pieces = total < A.blocks ? total : A.blocks;
        if (w >= pieces) {
            if (threadIdx.x == 0) span[0] = 0;
            return;
        }
        pg_i64 x = total * w / pieces;
        const pg_i64 x1 = total * (w + 1) / pieces;
        if (x >= before && x < before + sum) {
            pg_i64 at = before;
            for (pg_i64 b = b0; b < b1; ++b) {
                const Request r = request(A, b, false);
                const pg_i64 items = static_cast<pg_i64>(A.heads) * r.units * r.kt;
                if (x < at + items) {
                    sh.begin[0] = b;
                    sh.begin[1] = at;
                    break;
                }
                at += items;
            }
        }
        __syncthreads();
        pg_i64 b = uniform64(sh.begin[0]), xb = uniform64(sh.begin[1]);
        int joined = 0;
        while (x < x1) {
            Request rq = request(A, b, false);
            rq.row = uniform(rq.row);
            rq.n = uniform(rq.n);
            rq.length = uniform(rq.length);
            rq.first = uniform(rq.first);
            rq.kt = uniform(rq.kt);
            rq.units = uniform(rq.units);
            const pg_i64 items = static_cast<pg_i64>(A.heads) * rq.units * rq.kt;
            if (x >= xb + items) {
                xb += items;
                ++b;
                continue;
            }
            const pg_i64 unit = (x - xb) / rq.kt;
            const int t0 = static_cast<int>(x - xb - unit * rq.kt);
            const int t1 = x1 - x < rq.kt - t0 ? t0 + static_cast<int>(x1 - x) : rq.kt;
            const int h = static_cast<int>(unit / rq.units), in = static_cast<int>(unit - static_cast<pg_i64>(h) * rq.units);
            const int tile = in / HS, hs = in - tile * HS;
            Unit u;
            u.table = A.table + b * A.s_table;
            u.aim(A, h);
            u.n = rq.n - tile * C < C ? rq.n - tile * C : C;
            u.p0 = rq.length - rq.n + tile * C;
            u.hi = u.p0 + u.n > 0 ? u.p0 + u.n : 0;
            u.lo = 0;
            if (WIN && u.p0 + 1 > A.window) u.lo = u.p0 + 1 - A.window;
            const int row = rq.row + tile * C, head = h * G + hs * RB;
            State st;
            load_q(A, u, row, head, st);
            piece<kAttendTile>(A, u, (rq.first + t0) * kAttendTile + 32 * wave, (rq.first + t1) * kAttendTile, st);
            // The four waves' results.
            const int lane = own_lane(), n = lane & 15, g = lane >> 4;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                st.l[t] = over_groups(st.l[t], [](float a, float b) { return a + b; });
                if (g == 0) {
                    sh.m[wave][16 * t + n] = st.m[t];
                    sh.l[wave][16 * t + n] = st.l[t];
                }
            }
            __syncthreads();
            float m[NT], l[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                m[t] = -__builtin_inff();
#pragma unroll
                for (int k = 0; k < 4; ++k) m[t] = fmaxf(m[t], sh.m[k][16 * t + n]);
                l[t] = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float mk = sh.m[k][16 * t + n];
                    l[t] += mk == -__builtin_inff() ? 0.0f : sh.l[k][16 * t + n] * __builtin_amdgcn_exp2f(mk - m[t]);
                }
                const float f = st.m[t] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(st.m[t] - m[t]);
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) sh.o[wave][(t * NK + j) * 4 + q][lane] = st.o[t][j][q] * f;
            }
            __syncthreads();
            const bool opens = t0 == 0, closes = t1 == rq.kt;
            float* const part = A.parts + (2 * w + (opens ? 1 : 0)) * PART;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int r = 16 * t + n, i = r / GH, hh = r - i * GH;
                const bool valid = i < u.n && (HS == 1 || hs * RB + hh < G);
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    if ((t * NK + j) % 4 != wave) continue;
                    pg_f32x4 o[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        o[q] = sh.o[0][(t * NK + j) * 4 + q][lane];
#pragma unroll
                        for (int k = 1; k < 4; ++k) o[q] += sh.o[k][(t * NK + j) * 4 + q][lane];
                    }
                    if (!valid) continue;
                    if (opens && closes) {
                        write_row(A, row + i, head + hh, g, j, o, l[t] == 0.0f ? 0.0f : 1.0f / l[t]);
                    } else {
                        float* const po = part + 2 * RB + r * DP + 64 * j + 16 * g;
#pragma unroll
                        for (int e = 0; e < 4; ++e) *reinterpret_cast<pg_f32x4*>(po + 4 * e) = pg_f32x4{o[0][e], o[1][e], o[2][e], o[3][e]};
                    }
                }
                if (wave == 0 && g == 0 && valid) {
                    if (!(opens && closes)) {
                        part[r] = m[t];
                        part[RB + r] = l[t];
                    } else if (LSE) {
                        A.lse[(row + i) * A.s_lse[0] + (head + hh) * A.s_lse[1]] = lse_of(m[t], l[t]);
                    }
                }
            }
            if (opens && !closes) {
                joined = 1;
                if (threadIdx.x == 0) {
                    // The workgroup of the unit's last item.
                    const pg_i64 last = xb + (unit + 1) * rq.kt - 1;
                    span[1] = row;
                    span[2] = head;
                    span[3] = u.n;
                    span[4] = static_cast<int>(((last + 1) * pieces - 1) / total);
                    span[5] = hs;
                }
            }
            x += t1 - t0;
        }
        if (threadIdx.x == 0) span[0] = joined;
    }

    __device__ static float lse_of(float m, float l) {
        return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
    }

    // This wave's steps of 32 tokens from `base` on, STRIDE tokens apart, below
    // `end`.  The next step's pages and bytes are under way during one.
    template <int STRIDE>
    __device__ static void piece(const AttendArgs& A, const Unit& u, int base, int end, State& st) {
        if (end > u.hi) end = u.hi;
        if (base + 32 <= u.lo) base += (u.lo - base - 32 + STRIDE) / STRIDE * STRIDE;
        if (base >= end) return;
        // Page numbers are on their way before the bytes of the step ahead, so that
        // waiting for them is not waiting for those.
        Pages pg, ahead;
        Raw a, b;
        pages(A, u, base, pg);
        pages(A, u, base + STRIDE, ahead);
        load(A, u, base, pg, a);
        for (;;) {
            if (base + STRIDE < end) {
                pg = ahead;
                pages(A, u, base + 2 * STRIDE, ahead);
                load(A, u, base + STRIDE, pg, b);
            }
            step(A, u, base, a, st);
            base += STRIDE;
            if (base >= end) return;
            if (base + STRIDE < end) {
                pg = ahead;
                pages(A, u, base + 2 * STRIDE, ahead);
                load(A, u, base + STRIDE, pg, a);
            }
            step(A, u, base, b, st);
            base += STRIDE;
            if (base >= end) return;
        }
    }
    // ---- prompts ----
    // A unit is 4 * C tokens, C for each wave of a workgroup: the waves read the
    // same keys at about the same time, each for rows of its own, and need not
    // meet.  list_units() lists the units, the longest first, those beyond 1.3 of
    // a workgroup's share of the work in several pieces, which finish() joins in
    // the launch behind.
    static constexpr int kUnitTokens = 4 * C;

    struct Span {
        int lo, hi;  // tokens of a unit's keys, lo a multiple of 32
    };
    __device__ static Span span_of(const AttendArgs& A, const Request& rq, int tile) {
        const int p0 = rq.length - rq.n + tile * kUnitTokens;
        const int n = rq.n - tile * kUnitTokens < kUnitTokens ? rq.n - tile * kUnitTokens : kUnitTokens;
        Span s;
        s.hi = p0 + n > 0 ? p0 + n : 0;
        s.lo = WIN && p0 + 1 > A.window ? (p0 + 1 - A.window) / 32 * 32 : 0;
        return s;
    }

    // units: {entries, pieces to be done over, units in several pieces}, then
    // entries {request, tile, piece << 16 | pieces, first partial result}; behind
    // the room for them a counter for each partial result (zeroed here), the
    // pieces to be done over, and the first pieces of units in several.
    template <int THREADS>
    __device__ static void list_units(const AttendArgs& A) {
        constexpr int BUCKETS = 128;
        __shared__ pg_i64 lds[THREADS / 64];
        __shared__ int many[BUCKETS], slots, cuts;
        __shared__ pg_u64 work;
        const pg_i64 per = (A.batch + THREADS - 1) / THREADS, b0 = threadIdx.x * per;
        const pg_i64 b1 = b0 + per < A.batch ? b0 + per : A.batch;
        if (threadIdx.x < BUCKETS) many[threadIdx.x] = 0;
        if (threadIdx.x == 0) {
            slots = 0;
            cuts = 0;
            work = 0;
            A.units[1] = 0;
            A.units[2] = 0;
        }
        int* const count = A.units + kUnitHead + A.room * kUnitInts;
        for (int i = threadIdx.x; i < A.counters; i += THREADS) count[i] = 0;
        __shared__ pg_i64 before[THREADS];
        pg_i64 units = 0, total;
        // With a request out of range the rest may add up to more rows than there
        // are, and than the list has room for: the list stays empty then.
        constexpr pg_i64 kBad = pg_i64(1) << 40;
        bool bad = false;
        for (pg_i64 b = b0; b < b1; ++b) {
            const Request rq = request(A, b, false);
            bad |= rq.bad;
            units += (rq.n + kUnitTokens - 1) / kUnitTokens;
        }
        before[threadIdx.x] = block_scan<THREADS>(bad ? kBad : units, total, lds);
        __syncthreads();
        if (total >= kBad) {
            if (threadIdx.x == 0) {
                A.units[0] = 0;
                *A.err = 7;
            }
            return;
        }
        // Three passes over the units, spread over the threads: the work, the
        // sizes, the places.
        int limit = 0x7FFFFFFF;
        float per_step = 0.0f;
        struct Listed {
            int b, tile, steps;
        };
        auto find = [&](pg_i64 i) {
            int lo = 0, hi = THREADS;  // before[lo] <= i < before[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (before[mid] <= i) lo = mid;
                else hi = mid;
            }
            pg_i64 b = lo * per, at = before[lo];
            Request rq = request(A, b, false);
            for (;;) {
                const int tiles = (rq.n + kUnitTokens - 1) / kUnitTokens;
                if (i < at + tiles) break;
                at += tiles;
                rq = request(A, ++b, false);
            }
            const Span s = span_of(A, rq, static_cast<int>(i - at));
            return Listed{static_cast<int>(b), static_cast<int>(i - at), s.hi > s.lo ? (s.hi - s.lo + 31) / 32 : 1};
        };
        Listed own{};  // this thread's first unit
        if (threadIdx.x < total) own = find(threadIdx.x);
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            pg_u64 sum = 0;
            for (pg_i64 i = threadIdx.x; i < total; i += THREADS) {
                const Listed unit = i < THREADS ? own : find(i);
                const int tile = unit.tile, steps = unit.steps;
                sum += static_cast<pg_u64>(steps);
                if (pass == 0) continue;
                const int pieces = (steps + limit - 1) / limit, size = steps < limit ? steps : limit;
                const int bucket = BUCKETS - 1 - static_cast<int>(static_cast<float>(size) * per_step);
                const int place = atomicAdd(&many[bucket], pieces * HS);
                if (pass == 1) continue;
                for (int hs = 0; hs < HS; ++hs) {
                    const int slot = pieces > 1 ? atomicAdd(&slots, pieces) : 0;
                    if (pieces > 1) cut(A)[atomicAdd(&cuts, 1)] = place + hs * pieces;
                    for (int k = 0; k < pieces; ++k) {
                        int* const e = A.units + kUnitHead + static_cast<pg_i64>(place + hs * pieces + k) * kUnitInts;
                        e[0] = unit.b;
                        e[1] = tile * HS + hs;
                        e[2] = k << 16 | pieces;
                        e[3] = slot;
                    }
                }
            }
            if (pass == 0) atomicAdd(&work, sum);
            __syncthreads();
            if (pass == 0) {
                // 1.3 of a workgroup's share, above 1 so that the pieces are bounded: chunks
                // over cached contexts 251 us at 1.05, 245 at 1.2, 217 at 1.3; 512 tokens over
                // 32768 364 at 1.3, 431 at 1.4.
                const float share = static_cast<float>(work) * (1.3f * HS * A.heads / A.cus);
                limit = share < 16.0f ? 16 : share > 0x7FFFF00 ? 0x7FFFF00 : static_cast<int>(share) + 1;
                per_step = (BUCKETS - 1) / (static_cast<float>(limit) * 1.0001f);  // below BUCKETS - 1 for a whole one
            } else if (pass == 1) {
                // Places of the buckets, longest units first.
                pg_i64 entries;
                const int first = static_cast<int>(block_scan<THREADS>(threadIdx.x < BUCKETS ? many[threadIdx.x] : 0, entries, lds));
                if (threadIdx.x == 0) A.units[0] = static_cast<int>(entries);
                if (threadIdx.x < BUCKETS) many[threadIdx.x] = first;
            }
            __syncthreads();
        }
        if (threadIdx.x == 0) A.units[2] = cuts;
    }

    // A piece of a unit, as one wave of a workgroup sees it.
    struct Part {
        int b, h, tile, hs, piece, pieces, slot;
        int base, end;   // tokens of the piece
        int row, head;   // of the wave's rows
        Request rq;
        Unit u;
    };
    __device__ static void part_of(const AttendArgs& A, int entry, int h, Part& p) {
        const int wave = uniform(threadIdx.x >> 6);
        p.h = h;
        const int* const e = A.units + kUnitHead + static_cast<pg_i64>(entry) * kUnitInts;
        const int code = uniform(e[1]), kp = uniform(e[2]);
        p.b = uniform(e[0]);
        p.slot = uniform(e[3]);
        p.piece = static_cast<int>(static_cast<pg_u32>(kp) >> 16);
        p.pieces = kp & 0xFFFF;
        p.tile = code / HS;
        p.hs = code - p.tile * HS;
        p.rq = request(A, p.b, true);
        p.rq.row = uniform(p.rq.row);
        p.rq.n = uniform(p.rq.n);
        p.rq.length = uniform(p.rq.length);
        const Span s = span_of(A, p.rq, p.tile);
        const int steps = s.hi > s.lo ? (s.hi - s.lo + 31) / 32 : 1;
        p.base = s.lo + 32 * static_cast<int>(static_cast<pg_i64>(steps) * p.piece / p.pieces);
        p.end = s.lo + 32 * static_cast<int>(static_cast<pg_i64>(steps) * (p.piece + 1) / p.pieces);
        if (p.end > s.hi) p.end = s.hi;
        const int first = p.tile * kUnitTokens + wave * C;
        p.row = p.rq.row + first;
        p.head = p.h * G + p.hs * RB;
        p.u.table = A.table + p.b * A.s_table;
        p.u.h = p.h;
        p.u.n = p.rq.n - first < C ? p.rq.n - first : C;
        p.u.p0 = p.rq.length - p.rq.n + first;
        p.u.hi = p.u.n > 0 && p.u.p0 + p.u.n > 0 ? p.u.p0 + p.u.n : 0;
        p.u.lo = WIN && p.u.p0 + 1 > A.window ? p.u.p0 + 1 - A.window : 0;
    }
    __device__ static float* part_sums(const AttendArgs& A, const Part& p, int piece) {
        const int wave = uniform(threadIdx.x >> 6);
        return A.unit_parts + ((static_cast<pg_i64>(p.slot + piece) * A.heads + p.h) * 4 + wave) * PART;
    }

    // Place of a unit's row (token, head of the group) in a partial result.
    __device__ static int place_of(int i, int hh) { return HS == 1 ? i * G + hh : hh % RB; }

    // The steps of a wave's rows, by itself, 16 * NT rows at a time.  The piece
    // is one of W's, whose units may be wider.
    template <class W>
    __device__ static void rows(const AttendArgs& A, const typename W::Part& p) {
        const int heads = W::HS == 1 ? G : (G - p.hs * W::RB < W::RB ? G - p.hs * W::RB : W::RB);
#pragma unroll 1
        for (int i0 = 0; i0 < p.u.n; i0 += C)
#pragma unroll 1
            for (int h0 = 0; h0 < heads; h0 += GH) {
                Unit u;
                u.table = p.u.table;
                u.aim(A, p.h);
                u.n = p.u.n - i0 < C ? p.u.n - i0 : C;
                u.p0 = p.u.p0 + i0;
                u.hi = u.p0 + u.n > 0 ? u.p0 + u.n : 0;
                u.lo = WIN && u.p0 + 1 > A.window ? u.p0 + 1 - A.window : 0;
                const int row = p.row + i0, head = p.head + h0;
                State st;
                load_q(A, u, row, head, st);
                piece<32>(A, u, p.base, p.end, st);
                const int lane = own_lane(), n = lane & 15, g = lane >> 4;
                float* const part = W::part_sums(A, p, p.piece);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    st.l[t] = over_groups(st.l[t], [](float a, float b) { return a + b; });
                    const int r = 16 * t + n, i = r / GH, hh = r - i * GH;
                    if (i >= u.n || h0 + hh >= heads) continue;
                    if (p.pieces == 1) {
                        const float f = st.l[t] == 0.0f ? 0.0f : 1.0f / st.l[t];
#pragma unroll
                        for (int j = 0; j < NK; ++j) write_row(A, row + i, head + hh, g, j, st.o[t][j], f);
                        if (LSE && g == 0) A.lse[(row + i) * A.s_lse[0] + (head + hh) * A.s_lse[1]] = lse_of(st.m[t], st.l[t]);
                    } else {
                        const int at = W::place_of(i0 + i, h0 + hh);
                        if (g == 0) {
                            part[at] = st.m[t];
                            part[W::RB + at] = st.l[t];
                        }
#pragma unroll
                        for (int j = 0; j < NK; ++j)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                *reinterpret_cast<pg_f32x4*>(part + 2 * W::RB + at * DP + 64 * j + 16 * g + 4 * k) =
                                    pg_f32x4{st.o[t][j][0][k], st.o[t][j][1][k], st.o[t][j][2][k], st.o[t][j][3][k]};
                    }
                }
            }
    }

    // Joins the pieces of a unit, in the launch behind theirs: by the last piece to
    // end it takes fences, which write back and empty whole L2 caches (chunks over
    // cached contexts 307 us, so 240).
    __device__ static int* counter(const AttendArgs& A, const Part& p) {
        return A.units + kUnitHead + A.room * kUnitInts + p.slot * A.heads + p.h;
    }
    __device__ static void join_pieces(const AttendArgs& A, const Part& p) {
        const int lane = threadIdx.x & 63;
        if (p.u.n <= 0) return;
        // Lane r < RB weighs row r; the lanes share the rows' numbers, four each.
        constexpr int LANES = DP / 4, AT_ONCE = 64 / LANES, TURNS = RB / AT_ONCE;
        const pg_i64 next = static_cast<pg_i64>(A.heads) * 4 * PART;
        const float* const part = part_sums(A, p, 0);
        const int sub = lane / LANES, d = 4 * (lane - sub * LANES), r = lane & (RB - 1);
        float m = -__builtin_inff(), l = 0.0f;
        auto valid = [&](int row) {
            const int i = row / GH, hh = row - i * GH;
            return i < p.u.n && i < C && (HS == 1 || p.hs * RB + hh < G);
        };
        if (valid(r))
            for (int k = 0; k < p.pieces; ++k) m = fmaxf(m, part[k * next + r]);
        pg_f32x4 o[TURNS];
#pragma unroll
        for (int t = 0; t < TURNS; ++t) o[t] = pg_f32x4{0, 0, 0, 0};
        for (int k = 0; k < p.pieces; ++k) {
            float w = 0.0f;
            if (valid(r)) {
                const float mk = part[k * next + r];
                w = mk == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mk - m);
                l += w * part[k * next + RB + r];
            }
#pragma unroll
            for (int t = 0; t < TURNS; ++t) {
                const int row = t * AT_ONCE + sub;
                const float f = __shfl(w, row, 64);
                if (valid(row)) o[t] += f * *reinterpret_cast<const pg_f32x4*>(part + k * next + 2 * RB + row * DP + d);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
            const int row = t * AT_ONCE + sub;
            const float f = __shfl(inv, row, 64);
            if (!valid(row) || d >= D) continue;
            const int i = row / GH, hh = row - i * GH;
            char* const q = A.out + ((p.row + i) * A.s_out[0] + (p.head + hh) * A.s_out[1] + d) * elem_size(QT);
#pragma unroll
            for (int e = 0; e < 4; ++e) store_elem<QT>(q + e * elem_size(QT), o[t][e] * f);
        }
        if (LSE && lane < RB && valid(r)) {
            const int i = r / GH, hh = r - i * GH;
            A.lse[(p.row + i) * A.s_lse[0] + (p.head + hh) * A.s_lse[1]] = lse_of(m, l);
        }
    }

    // ---- prompts, tile by tile ----
    // The four waves convert a tile of 64 tokens once, 16 each, into LDS: keys
    // as rows of bf16 (f16 for f16 queries), values as columns of f16, both in
    // the order in which v_mfma_f32_32x32x16 takes them, two tiles in turn with
    // one barrier a tile.  A wave has 32 query rows: lane (n, h) of 32 x 2 holds
    // of row n tokens 8k + 4h .. + 3 of the scores, which are the P operand.
    // p enters as f16: between 2^10 and 2^14 at a row's maximum (kLift, kLag), so
    // that no p that matters is subnormal; in one part for bf16 outputs (2^-11 of
    // it, as much again of each value and of its scale), in two for f16 ones.
    // Values are relative to a base that follows the pages' scales (kLow, kHigh:
    // as f16 values, no code of theirs is too large or loses more than one of a
    // scale's 2^8; f16 outputs have the scales in p); where those spread too far
    // for f16, or a NaN lies among values that some rows do not
    // see, the waves do the piece over with bf16 parts (rows).
    static constexpr bool TILES = PROMPT && NT == 2 && PAGED16 && D <= 128 && QT != kF32;
    static constexpr int kTile = 64, kChunks = DP / 8;  // tokens; 16-byte pieces of a key
    static constexpr float kLift = 10.0f, kLag = 4.0f;
    static constexpr int TP = QT == kF16 ? 2 : 1;       // parts of p
    static constexpr float kLow = TP == 1 ? 0x1p-8f : 0x1p-5f, kHigh = TP == 1 ? 0x1p6f : 2.0f, kStart = TP == 1 ? 0x1p-4f : 1.0f;

    // LDS: {keys, values} of one tile, then of the next.  A key is a row of
    // kChunks 16-byte pieces, a value's dimension one of 8 (64 tokens); a piece
    // lies where the exclusive or of its number and a function of its row says, so
    // that neither the waves' writes nor the MFMAs' reads meet in a bank more
    // often than their size asks, and a lane's addresses differ in few bits.
    static constexpr int kRow = 2 * DP, kPart = kTile * kRow, kBuffer = 2 * kPart;
    struct Tiles {
        alignas(1024) char bytes[2 * kBuffer];
        float ks[4][4], vs[4][4];  // scales of four tiles in turn, one for each 16 tokens
        int bad[2];
    };
    __device__ static int key_bits(int token) { return kChunks == 16 ? token & 15 : token >> 1 & 7; }
    __device__ static int value_bits(int d) { return (d >> 1 & 7) ^ (d >> 4 & 1); }

    struct Stage {
        pg_u32x4 k[kChunks / 8];
        pg_u32 v[8];
    };
    // Positions that the unit's rows attend to, together.
    struct Reach {
        int lo, hi;
    };
    // Loads that all lanes share, as vector loads: they return in order, where
    // scalar ones make every wait for LDS wait for them too.
    template <class T>
    __device__ static T shared_load(const T* p) {
        int zero = 0;
        asm volatile("" : "+v"(zero));
        return p[zero];
    }
    // The page of this wave's 16 tokens of the tile at `base`.
    __device__ static int tile_page(const AttendArgs& A, const Part& p, const Reach& r, int base) {
        int t = base + 16 * uniform(threadIdx.x >> 6);
        t = t < r.lo ? r.lo : t >= r.hi ? r.hi - 1 : t;
        return shared_load(p.u.table + static_cast<pg_u32>(t) / PAGE);
    }
    // Pieces behind the head size repeat the last one, as in load().
    __device__ static void tile_load(const AttendArgs& A, const Part& p, int base, int id, Stage& s) {
        const int lane = threadIdx.x & 63;
        const int off = static_cast<int>(static_cast<pg_u32>(base + 16 * uniform(threadIdx.x >> 6)) % PAGE);
        const char* const kp = A.cache[0] + id * A.s_cache[0][0] + p.h * A.s_cache[0][1] + off * A.s_cache[0][2];
        const char* const vp = A.cache[1] + id * A.s_cache[1][0] + p.h * A.s_cache[1][1] + off * A.s_cache[1][2];
        const int kd = (lane & 3) * (DP / 4), ko = (lane >> 2) * static_cast<int>(A.s_cache[0][2]);
#pragma unroll
        for (int j = 0; j < kChunks / 8; ++j)
            s.k[j] = *reinterpret_cast<const pg_u32x4*>(kp + ko + (D % 64 != 0 && kd + 16 * j > D - 16 ? D - 16 : kd + 16 * j));
        const int vd = 4 * (lane & (DP / 4 - 1)), h = value_half(lane), vt = static_cast<int>(A.s_cache[1][2]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s.v[i] = *reinterpret_cast<const pg_u32*>(vp + (4 * h + (i & 3) + 2 * (i & 4)) * vt + (D % 64 != 0 && vd > D - 4 ? D - 4 : vd));
    }
    // Which half of the tokens a lane's values are of; up to head size 64 the
    // upper lanes repeat the lower ones'.
    __device__ static int value_half(int lane) { return lane / (DP / 4) & 1; }

    // A tile that some row does not see whole: what lies outside the unit's
    // positions may be anything.
    __device__ static void tile_edge(const Reach& r, Stage& s, int base, Tiles& T, int buf) {
        const int wave = uniform(threadIdx.x >> 6), h = value_half(own_lane());
        pg_u32 nan = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = base + 16 * wave + 4 * h + (i & 3) + 2 * (i & 4);
            s.v[i] = at >= r.lo && at < r.hi ? s.v[i] : 0;
            nan |= ((s.v[i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
        }
        if (CT == kE4M3 && nan) T.bad[buf] = 1;
    }

    // The conversion of a wave's tokens, in kWrites steps of one LDS write each.
    // w: the values' scale relative to the base (f16 outputs: p takes it).
    static constexpr int kWrites = kChunks / 4 + 4;
    __device__ static void tile_write(const Stage& s, _Float16 w, Tiles& T, int buf, int step) {
        const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
        if (step < kChunks / 4) {
            const int token = 16 * wave + (lane >> 2), i = step;
            const int ko = buf * kBuffer + token * kRow + (((lane & 3) * (kChunks / 4)) ^ key_bits(token)) * 16;
            const pg_u32 w0 = s.k[i >> 1][2 * (i & 1)], w1 = s.k[i >> 1][2 * (i & 1) + 1];
            *reinterpret_cast<pg_u32x4*>(T.bytes + (ko ^ 16 * i)) =
                pg_u32x4{codes2<CT, H, false>(w0), codes2<CT, H, true>(w0), codes2<CT, H, false>(w1), codes2<CT, H, true>(w1)};
            return;
        }
        const int d = 4 * (lane & (DP / 4 - 1)), h = lane / (DP / 4), q = step - kChunks / 4;
        const int vo = buf * kBuffer + kPart + d * 128 + ((2 * wave + h) ^ value_bits(d)) * 16;
        pg_u32x4 out;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const pg_u32 a = __builtin_amdgcn_perm(s.v[2 * e + 1], s.v[2 * e], q < 2 ? 0x05010400u : 0x07030602u);
            const pg_u32 x = q & 1 ? codes2<CT, true, true>(a) : codes2<CT, true, false>(a);
            out[e] = TP == 1 ? __builtin_bit_cast(pg_u32, __builtin_bit_cast(pg_h2, x) * pg_h2{w, w}) : x;
        }
        if (DP == 128 || h < 2) *reinterpret_cast<pg_u32x4*>(T.bytes + (vo ^ 16 * (q >> 1)) + 128 * q) = out;
    }

    __device__ static pg_f32x16 mma32(pg_u32x4 a, pg_u32x4 b, pg_f32x16 c, bool half) {
        if (half) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pg_h8, a), __builtin_bit_cast(pg_h8, b), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pg_bf8, a), __builtin_bit_cast(pg_bf8, b), c, 0, 0, 0);
    }

    // False where the piece is to be done over.
    __device__ static bool tiles(const AttendArgs& A, const Part& p, Tiles& T) {
        constexpr int KS = DP / 16, DT = DP / 32;
        const int lane = own_lane(), n = lane & 31, h = lane >> 5, wave = uniform(threadIdx.x >> 6);
        const int row_i = n / GH, row_h = n - row_i * GH;
        const auto has_row = [&](int i, int hh) { return i < p.u.n && i < C && (HS == 1 || p.hs * RB + hh < G); };
        const bool valid = has_row(row_i, row_h);
        // The lane's row attends to positions lo .. hi - 1; all the unit's rows to
        // those of every tile between `from` and `till`.
        const int hi = p.u.p0 + row_i + 1 < p.end ? p.u.p0 + row_i + 1 : p.end;
        const int lo = WIN ? p.u.p0 + row_i + 1 - A.window : 0;
        const int first = p.rq.length - p.rq.n + p.tile * kUnitTokens;  // position of the unit's first row
        const int ntok = p.rq.n - p.tile * kUnitTokens < kUnitTokens ? p.rq.n - p.tile * kUnitTokens : kUnitTokens;
        const int till = first + 1 < p.end ? first + 1 : p.end, from = WIN ? first + ntok - A.window : 0;
        Reach reach;
        reach.hi = first + ntok < p.end ? first + ntok : p.end;
        reach.lo = WIN && first + 1 > A.window ? first + 1 - A.window : 0;
        // q, with the sign of `factor`: scores are products with scales >= 0.
        const pg_u32 flip = A.factor < 0.0f ? 0x80008000u : 0u;
        const float factor = fabsf(A.factor);
        pg_u32x4 q[KS];
        // Places without a row or a dim read the unit's first row, or a dim inside, and are 0.
        const char* const qp = A.q + (static_cast<pg_i64>(valid ? p.row + row_i : p.rq.row + p.tile * kUnitTokens) * A.s_q[0] +
                                      (p.head + (valid ? row_h : 0)) * A.s_q[1]) * 2;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            const int d = 16 * j + 8 * h;
            const bool in = valid && (D % 64 == 0 || d < D);
            Eight<QT> x8;
            load8<QT, VEC>(qp + (D % 64 != 0 && d >= D ? D - 8 : d) * 2, x8);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[j][e] = (in ? x8.w[e] : 0) ^ flip;
        }
        pg_f32x16 o[DT];
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        float m = -__builtin_inff(), l = 0.0f;
        float unit = 1.0f, next = 1.0f;  // base of the sums, and of the tile that is converted next
        bool done = true;
        if (reach.hi > p.base) {
            float ks, vs;  // of this wave's tokens two tiles ahead
            auto scales = [&](int id) {
                ks = shared_load(A.scale[0] + id * A.s_scale[0][0] + p.h * A.s_scale[0][1]);
                vs = shared_load(A.scale[1] + id * A.s_scale[1][0] + p.h * A.s_scale[1][1]);
            };
            auto post = [&](int slot) {
                if (lane == 0) {
                    T.ks[slot][wave] = ks;
                    T.vs[slot][wave] = vs;
                }
            };
            auto four = [&](const float* v) { return *reinterpret_cast<const pg_f32x4*>(v); };
            auto frag = [&](int at) { return *reinterpret_cast<const pg_u32x4*>(T.bytes + at); };
            // Whether a tile's values suit f16 relative to a base, which moves if need be.
            float inv = 1.0f;  // 1 / next
            auto settle = [&](const pg_f32x4 v) -> bool {
                const float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), low = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
                if (__ballot(!(top <= next * kHigh && low >= next * kLow))) {
                    next = top * kStart;
                    inv = 1.0f / next;
                    return __ballot(!(next <= 0x1p36f && next >= 0x1p-36f && low >= next * kLow)) == 0;
                }
                return true;
            };
            auto edge_of = [&](int base) { return base + kTile > till || base < from; };
            Stage s;
            // Two tiles' scales and the first one's bytes, then the second's.
            int id = checked(A, uniform(tile_page(A, p, reach, p.base)));
            tile_load(A, p, p.base, id, s);
            scales(id);
            if (threadIdx.x < 2) T.bad[threadIdx.x] = 0;
            post(0);
            id = checked(A, uniform(tile_page(A, p, reach, p.base + kTile)));
            scales(id);
            post(1);
            int id2 = checked(A, uniform(tile_page(A, p, reach, p.base + 2 * kTile))), id3 = tile_page(A, p, reach, p.base + 3 * kTile);
            __syncthreads();
            done = settle(four(T.vs[0]));
            if (edge_of(p.base)) tile_edge(reach, s, p.base, T, 0);
            if (done) {
                const _Float16 w = static_cast<_Float16>(T.vs[0][wave] * inv);
#pragma unroll
                for (int i = 0; i < kWrites; ++i) tile_write(s, w, T, 0, i);
            }
            if (done) {
                if (p.base + kTile < reach.hi) tile_load(A, p, p.base + kTile, id, s);
                scales(id2);
                __syncthreads();
                int buf = 0, slot = 0;
                // Where the lane's first pieces of a key and a value lie.
                const int k0 = n * kRow + (h ^ key_bits(n)) * 16, v0 = kPart + n * 128 + (h ^ value_bits(n)) * 16;
                for (int base = p.base;; base += kTile, buf ^= 1, slot = (slot + 1) & 3) {
                    const bool edge = edge_of(base), more = base + kTile < reach.hi;
                    if (CT == kE4M3 && edge && uniform(T.bad[buf])) {
                        done = false;
                        break;
                    }
                    if (__ballot(next != unit)) {
                        const float f = unit / next;
#pragma unroll
                        for (int t = 0; t < DT; ++t) o[t] *= f;
                        unit = next;
                    }
                    const float wnext = T.vs[(slot + 1) & 3][wave];
                    if (more) {
                        done = settle(four(T.vs[(slot + 1) & 3]));
                        if (!done) break;
                        if (edge_of(base + kTile)) tile_edge(reach, s, base + kTile, T, buf ^ 1);
                    }
                    // Scores of the two halves of the tile, their keys read half a tile
                    // ahead; beside the MFMAs the next tile's conversion into the other
                    // buffer, whose last readers have passed the barrier (after the last
                    // tile: of anything).  The order is kept as it stands here.
                    const int kb = k0 + buf * kBuffer, vb = v0 + buf * kBuffer;
                    const _Float16 wh = static_cast<_Float16>(wnext * inv);
                    pg_f32x16 x[2];
                    pg_u32x4 kf[KS], vf[DT];
#pragma unroll
                    for (int j = 0; j < KS; ++j) kf[j] = frag(kb ^ 32 * j);
                    pg_f32x4 f = four(T.ks[slot]) * factor;
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int j = 0; j < KS; ++j) {
                            pg_f32x16 zero;
#pragma unroll
                            for (int i = 0; i < 16; ++i) zero[i] = 0.0f;
                            x[a] = mma32(kf[j], q[j], j ? x[a] : zero, H);
                            if (a == 0) kf[j] = frag((kb ^ 32 * j) + 32 * kRow);
                            else if (j < DT) vf[j] = frag(vb + 4096 * j);
#pragma unroll
                            for (int i = (a * KS + j) * kWrites / (2 * KS); i < (a * KS + j + 1) * kWrites / (2 * KS); ++i) tile_write(s, wh, T, buf ^ 1, i);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    if (edge) {
#pragma unroll
                        for (int a = 0; a < 2; ++a)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int at = base + 32 * a + 8 * (i >> 2) + 4 * h + (i & 3);
                                x[a][i] = at < hi && at >= lo ? x[a][i] * f[2 * a + (i >> 3)] : -__builtin_inff();
                            }
                        f = pg_f32x4{1.0f, 1.0f, 1.0f, 1.0f};
                    }
                    float mx[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mx[k] = x[k >> 1][8 * (k & 1)];
#pragma unroll
                        for (int i = 1; i < 8; ++i) mx[k] = fmaxf(mx[k], x[k >> 1][8 * (k & 1) + i]);
                    }
                    float peak = fmaxf(fmaxf(mx[0] * f[0], mx[1] * f[1]), fmaxf(mx[2] * f[2], mx[3] * f[3]));
                    if (__ballot(peak > m + (kLift + kLag))) {
                        peak = fmaxf(peak, __shfl_xor(peak, 32, 64));
                        const float to = fmaxf(m, peak - kLift), g = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
                        m = to;
                        l *= g;
#pragma unroll
                        for (int t = 0; t < DT; ++t) o[t] *= g;
                    }
                    const float ms = m == -__builtin_inff() ? 0.0f : m;
                    if (more) {
                        post((slot + 2) & 3);
                        const int ahead = checked(A, uniform(id3));  // loaded before the bytes: no wait for them
                        if (base + 2 * kTile < reach.hi) tile_load(A, p, base + 2 * kTile, id2, s);
                        id2 = ahead;
                        scales(id2);
                        id3 = tile_page(A, p, reach, base + 4 * kTile);
                    }
                    pg_f32x4 w;
                    if constexpr (TP > 1) w = four(T.vs[slot]) / unit;
                    // p of the next 16 tokens beside the MFMAs of these.
                    pg_u32x4 pk[2][TP];
                    auto weigh_two = [&](int k, int e) {
                        pg_f32x2 y;
#pragma unroll
                        for (int z = 0; z < 2; ++z) y[z] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[k >> 1][8 * (k & 1) + 2 * e + z], f[k], -ms));
                        if constexpr (TP > 1) {
                            l += y[0] + y[1];
                            float y0 = y[0] * w[k], y1 = y[1] * w[k];
                            // One value each for both parts: a conversion that takes in
                            // the product rounds the exact one, another the float32 one.
                            asm("" : "+v"(y0), "+v"(y1));
                            const pg_h2 c = __builtin_convertvector((pg_f32x2{y0, y1}), pg_h2);
                            pk[k & 1][0][e] = __builtin_bit_cast(pg_u32, c);
                            pk[k & 1][TP - 1][e] = __builtin_bit_cast(
                                pg_u32, __builtin_convertvector((pg_f32x2{y0 - static_cast<float>(c[0]), y1 - static_cast<float>(c[1])}), pg_h2));
                        } else {
                            const pg_h2 c = __builtin_convertvector(y, pg_h2);
                            pk[k & 1][0][e] = __builtin_bit_cast(pg_u32, c);
                            // The sum of the weights as they are used, so that their rounding cancels in part.
                            if constexpr (LSE) l += y[0] + y[1];
                            else l = __builtin_amdgcn_fdot2(c, pg_h2{static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)}, l, false);
                        }
                    };
#pragma unroll
                    for (int e = 0; e < 4; ++e) weigh_two(0, e);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int t = 0; t < DT; ++t) {
#pragma unroll
                            for (int z = 0; z < TP; ++z) o[t] = mma32(vf[t], pk[k & 1][z], o[t], true);
                            if (k < 3) {
                                vf[t] = frag((vb ^ 32 * (k + 1)) + 4096 * t);
#pragma unroll
                                for (int e = t * 4 / DT; e < (t + 1) * 4 / DT; ++e) weigh_two(k + 1, e);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    if (!more) break;
                    __syncthreads();
                }
            }
        }
        if (!done) return false;
        l += __shfl_xor(l, 32, 64);
        const int out_lane = own_lane(), out_n = out_lane & 31, out_h = out_lane >> 5, out_i = out_n / GH, out_hh = out_n - out_i * GH;
        if (!has_row(out_i, out_hh)) return true;
        const int at = p.row + out_i, head = p.head + out_hh;
        if (p.pieces == 1) {
            const float f = l == 0.0f ? 0.0f : unit / l;
            char* const op = A.out + (at * A.s_out[0] + head * A.s_out[1]) * 2;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 32 * t + 8 * i + 4 * out_h;
                    if (D % 64 != 0 && d >= D) continue;
                    if constexpr (VEC) {
                        pg_u32x2 w;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float a = o[t][4 * i + 2 * e] * f, b = o[t][4 * i + 2 * e + 1] * f;
                            if constexpr (QT == kF16) w[e] = __builtin_bit_cast(pg_u32, (pg_h2{static_cast<_Float16>(a), static_cast<_Float16>(b)}));
                            else w[e] = __builtin_bit_cast(pg_u32, __builtin_convertvector((pg_f32x2{a, b}), pg_bf2));
                        }
                        *reinterpret_cast<pg_u32x2*>(op + d * 2) = w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) store_elem<QT>(op + (d + e) * 2, o[t][4 * i + e] * f);
                    }
                }
            if (LSE && out_h == 0) A.lse[at * A.s_lse[0] + head * A.s_lse[1]] = lse_of(m, l);
        } else {
            float* const part = part_sums(A, p, p.piece);
            if (out_h == 0) {
                part[out_n] = m;
                part[RB + out_n] = l;
            }
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<pg_f32x4*>(part + 2 * RB + out_n * DP + 32 * t + 8 * i + 4 * out_h) =
                        pg_f32x4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]} * unit;
        }
        return true;
    }

    // Narrow: the kernel for 16 rows a wave.
    using Narrow = Attend<D, PAGE, G, 1, QT, CT, WIN, LSE, VEC, true>;
    __device__ static int* over(const AttendArgs& A) { return A.units + kUnitHead + A.room * kUnitInts + A.counters; }
    __device__ static int* cut(const AttendArgs& A) { return over(A) + A.room * A.heads; }

    __device__ static void prompt(const AttendArgs& A, Tiles& T) {
        const int entry = static_cast<int>(blockIdx.x / A.heads), h = static_cast<int>(blockIdx.x) - entry * A.heads;
        if (entry >= A.units[0]) return;
        Part p;
        part_of(A, entry, h, p);
        if constexpr (TILES) {
            if (!tiles(A, p, T) && threadIdx.x == 0) {
                over(A)[atomicAdd(A.units + 1, 1)] = static_cast<int>(blockIdx.x);
                if (p.pieces > 1) atomicAdd(counter(A, p), 1);
            }
        } else {
            Narrow::template rows<Attend>(A, p);
        }
    }

    // Prompts by the first workgroups, single tokens and few (F: the type for
    // those) by the last `blocks`.
    template <class F>
    __device__ static void both(const AttendArgs& A) {
        constexpr size_t few = sizeof(typename F::Shared), mine = TILES ? sizeof(Tiles) : 0;
        __shared__ __attribute__((aligned(1024))) char lds[few > mine ? few : mine];
        const int units = static_cast<int>(gridDim.x) - A.blocks;
        if (static_cast<int>(blockIdx.x) < units) prompt(A, *reinterpret_cast<Tiles*>(lds));
        else F::run(A, static_cast<int>(blockIdx.x) - units, *reinterpret_cast<typename F::Shared*>(lds));
    }

    // What remains: units that the workgroups for few rows left open, units in
    // several pieces, and pieces to be done over.
    template <class F>
    __device__ static void finish(const AttendArgs& A) {
        F::join(A);
        const int cuts = uniform(A.units[2]) * A.heads;
        for (int i = blockIdx.x; i < cuts; i += gridDim.x) {
            Part p;
            const int at = i / A.heads;
            part_of(A, uniform(cut(A)[at]), i - at * A.heads, p);
            // Low half: pieces to be done over, whose last one joins; high half: done.
            if ((uniform(*counter(A, p)) & 0xFFFF) == 0) join_pieces(A, p);
        }
        if constexpr (TILES) {
            __shared__ int arrived;
            const int many = uniform(A.units[1]);
            for (int i = blockIdx.x; i < many; i += gridDim.x) {
                const int at = uniform(over(A)[i]), entry = at / A.heads;
                Part p;
                part_of(A, entry, at - entry * A.heads, p);
                Narrow::template rows<Attend>(A, p);
                if (p.pieces == 1) continue;
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(counter(A, p), 0x10000, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
                const bool last = (arrived >> 16) + 1 == (arrived & 0xFFFF);
                __threadfence();
                if (last) join_pieces(A, p);
                __syncthreads();
            }
        }
    }

    // Joins the pieces of the unit that workgroup blockIdx.x left open.
    __device__ static void join(const AttendArgs& A) {
        constexpr int THREADS = 256, GROUPS = THREADS / RB;
        __shared__ float weight[THREADS], top[RB], sums[RB];
        __shared__ float red[GROUPS][RB];
        const int* const span = A.spans + static_cast<pg_i64>(blockIdx.x) * kSpanInts;
        if (!span[0]) return;
        const int row = span[1], head = span[2], ntok = span[3], last = span[4], hs = span[5];
        const int np = last - static_cast<int>(blockIdx.x) + 1;
        const int heads = HS == 1 ? GH : (G - hs * RB < RB ? G - hs * RB : RB), rows = HS == 1 ? ntok * GH : heads;
        auto part = [&](int k) { return A.parts + (2 * (static_cast<pg_i64>(blockIdx.x) + k) + (k == 0 ? 1 : 0)) * PART; };
        const int r = threadIdx.x % RB, grp = threadIdx.x / RB;
        float m = -__builtin_inff();
        if (r < rows)
            for (int k = grp; k < np; k += GROUPS) m = fmaxf(m, part(k)[r]);
        red[grp][r] = m;
        __syncthreads();
        if (threadIdx.x < RB) {
            for (int k = 1; k < GROUPS; ++k) m = fmaxf(m, red[k][r]);
            top[r] = m;
            sums[r] = 0.0f;
        }
        // Output pieces of four dims; the threads left over share the parts.
        constexpr int Q = DP / 4;
        const int pieces = rows * Q;
        float l = 0.0f;
        for (int p0 = 0; p0 < pieces; p0 += THREADS) {
            const int idx = p0 + static_cast<int>(threadIdx.x), pr = idx / Q, d = (idx - pr * Q) * 4;
            pg_f32x4 o = {0, 0, 0, 0};
            for (int k0 = 0; k0 < np; k0 += GROUPS) {
                // Weights of GROUPS parts.
                __syncthreads();
                const int k = k0 + grp;
                float wt = 0.0f;
                if (k < np && r < rows) {
                    const float mk = part(k)[r];
                    wt = mk == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mk - top[r]);
                    if (p0 == 0) l += wt * part(k)[RB + r];
                }
                weight[threadIdx.x] = wt;
                __syncthreads();
                if (idx < pieces) {
                    const int many = np - k0 < GROUPS ? np - k0 : GROUPS;
                    for (int k2 = 0; k2 < many; ++k2) {
                        const pg_f32x4 x = *reinterpret_cast<const pg_f32x4*>(part(k0 + k2) + 2 * RB + pr * DP + d);
                        o += x * weight[k2 * RB + pr];
                    }
                }
            }
            if (p0 == 0) {
                red[grp][r] = l;
                __syncthreads();
                if (threadIdx.x < RB) {
                    float s = 0.0f;
                    for (int k = 0; k < GROUPS; ++k) s += red[k][r];
                    sums[r] = s;
                }
                __syncthreads();
            }
            if (idx < pieces && d < D) {
                const int i = pr / GH, hh = pr - i * GH;
                const float s = sums[pr], f = s == 0.0f ? 0.0f : 1.0f / s;
                char* const p = A.out + ((row + i) * A.s_out[0] + (head + hh) * A.s_out[1] + d) * elem_size(QT);
#pragma unroll
                for (int e = 0; e < 4; ++e) store_elem<QT>(p + e * elem_size(QT), o[e] * f);
                if (LSE && d == 0) A.lse[(row + i) * A.s_lse[0] + (head + hh) * A.s_lse[1]] = lse_of(top[pr], s);
            }
        }
    }
};

}  // namespace ptowsp
