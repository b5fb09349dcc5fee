// k8_dev.h -- device helpers of the 8-bit dense layers.
#pragma once
#include "k8_gemm.h"

typedef __bf16 k8_bf16;
constexpr uint64_t k8_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }
constexpr int K8_CUS = 256;      // compute units of an MI355X: what a launch is sized for

// N values of T, 16 bytes or fewer, on T's own boundary: the memory system takes wide accesses at any address
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) K8Vec { T v[N]; };
template <class T, int N> __device__ __forceinline__ K8Vec<T, N> k8_load(const T *p) { return *(const K8Vec<T, N> *)p; }
template <class T, int N> __device__ __forceinline__ void k8_store(T *p, const K8Vec<T, N> &v) { *(K8Vec<T, N> *)p = v; }

typedef unsigned __attribute__((ext_vector_type(2), aligned(1))) k8_u32x2;
typedef unsigned __attribute__((ext_vector_type(4), aligned(1))) k8_u32x4;
typedef unsigned __attribute__((aligned(1))) k8_u32;
// rows of one launch where a workgroup or wavefront has a row: a grid holds fewer than 2^32 threads
constexpr int64_t K8_LAUNCH_ROWS = 1 << 23;
// results that are not read again soon: past the caches
template <class T, int N> __device__ __forceinline__ void k8_stream(T *p, const K8Vec<T, N> &v) {
    if constexpr (sizeof v == 16) { k8_u32x4 w; __builtin_memcpy(&w, &v, 16); __builtin_nontemporal_store(w, (k8_u32x4 *)p); }
    else if constexpr (sizeof v == 8) { k8_u32x2 w; __builtin_memcpy(&w, &v, 8); __builtin_nontemporal_store(w, (k8_u32x2 *)p); }
    else k8_store<T, N>(p, v);
}
// N numbers of T as the dwords they lie in: 16-bit numbers stay two to a register
template <class T, int N> struct K8Raw {
    unsigned w[N * sizeof(T) / 4];
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else if constexpr (__is_same(T, k8_bf16)) return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        else { typedef _Float16 h2 __attribute__((ext_vector_type(2))); return (float)__builtin_bit_cast(h2, w[e / 2])[e & 1]; }
    }
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, (const K8Vec<T, N> *)p, sizeof w); }
    // the first `have`, zeros behind them; p[have - 1] is the row's last number, even if p lies behind it.  No branch: a load in a branch of its own is waited for there
    __device__ __forceinline__ void load(const T *p, int have) {
        unsigned v[N];
#pragma unroll
        for (int e = 0; e < N; e++) {
            if constexpr (sizeof(T) == 4) v[e] = *(const unsigned *)(p + min(e, have - 1));
            else v[e] = *(const uint16_t *)(p + min(e, have - 1));
        }
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = e < have ? v[e] : 0u;
#pragma unroll
        for (int i = 0; i < (int)(sizeof w / 4); i++) {
            if constexpr (sizeof(T) == 4) w[i] = v[i];
            else w[i] = v[2 * i] | v[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void load(k8_global p) {
        if constexpr (sizeof w == 8) { const k8_u32x2 v = *(const __attribute__((address_space(1))) k8_u32x2 *)p; w[0] = v[0]; w[1] = v[1]; }
        else
#pragma unroll
            for (unsigned i = 0; i < sizeof w / 16; i++) {
                const k8_u32x4 v = *(const __attribute__((address_space(1))) k8_u32x4 *)(p + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; j++) w[4 * i + j] = v[j];
            }
    }
    __device__ __forceinline__ void load(k8_global p, int have) { load((const T *)(const char *)p, have); }
    // the largest magnitude; fp32: NaN does not count, 16 bits: it counts as infinity (two magnitudes are compared at a time, as whole numbers)
    __device__ __forceinline__ float most() const {
        if constexpr (sizeof(T) == 4) {
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < N; e++) m = fmaxf(m, fabsf(get(e)));
            return m;
        } else {
            typedef unsigned short u2 __attribute__((ext_vector_type(2)));
            u2 m = __builtin_bit_cast(u2, w[0] & 0x7fff7fffu);
#pragma unroll
            for (unsigned i = 1; i < sizeof w / 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u2, w[i] & 0x7fff7fffu));
            const unsigned t = m[0] > m[1] ? m[0] : m[1];
            if (t >= (__is_same(T, k8_bf16) ? 0x7f80u : 0x7c00u)) return __uint_as_float(0x7f800000u);
            K8Raw<T, 2> one = { { t } };
            return one.get(0);
        }
    }
    // the compiler knows nothing of what it computed from these registers before: it forms the values again instead of keeping them
    __device__ __forceinline__ void opaque() {
#pragma unroll
        for (unsigned i = 0; i < sizeof w / 4; i++) asm volatile("" : "+v"(w[i]));
    }
};

// the largest magnitude of a row, as the bit pattern of |x|: integers order like the magnitudes, and NaN and infinity sort above every number
__device__ __forceinline__ unsigned k8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
struct K8Scale { float r, s; };
__device__ __forceinline__ K8Scale k8_scale(unsigned top) {
    const float a = __uint_as_float(top);
    if (top >= 0x7f800000u) return { 0.0f, __uint_as_float(0x7fc00000u) };
    if (a < 0x1p-120f) return { 0.0f, 0.0f };
    return { 127.0f / a, a / 127.0f };
}
// rint(x r) as a byte.  Adding 1.5 2^23 leaves the rounded integer (to even) in the low mantissa bits, in two's complement; |x r| < 128.
// A row without a scale (r = 0) stores zeros whatever it holds
__device__ __forceinline__ unsigned k8_code(float x, float r) { return __float_as_uint(x * r + 12582912.0f) & 255u; }
__device__ __forceinline__ unsigned k8_codes(float x0, float x1, float x2, float x3, float r) {
    if (r == 0.0f) return 0u;
    const unsigned a = __float_as_uint(x0 * r + 12582912.0f), b = __float_as_uint(x1 * r + 12582912.0f);
    const unsigned c = __float_as_uint(x2 * r + 12582912.0f), d = __float_as_uint(x3 * r + 12582912.0f);
    const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return lo | hi << 16;
}
__device__ __forceinline__ float k8_relu(float v) { return v <= 0.0f ? 0.0f : v; }      // NaN stays
