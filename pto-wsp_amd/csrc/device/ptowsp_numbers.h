// Numbers of the operator kernels: element types, 8-bit codes, and pieces of eight elements.
#pragma once

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

}  // namespace ptowsp
