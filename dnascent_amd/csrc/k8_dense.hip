// k8_dense.hip -- 8-bit dense layers: rows in 8 bits, their product, its gradient (include/dnascent_hip.h has the formulas).
#include "k8_dense.h"
#include <stdint.h>

namespace {

typedef __bf16 bf16;

template <class T> __device__ __forceinline__ float k8_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T k8_to(float v) { return (T)v; }

// the largest magnitude of a row, as the bit pattern of |x|: integers order like the magnitudes, and NaN (0x7fc...) and infinity sort above every number
__device__ __forceinline__ unsigned k8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
struct RowScale { float r, s; };
__device__ __forceinline__ RowScale k8_scale(unsigned top) {
    const float a = __uint_as_float(top);
    if (top >= 0x7f800000u) return { 0.0f, __uint_as_float(0x7fc00000u) };
    if (a < 0x1p-120f) return { 0.0f, 0.0f };
    return { 127.0f / a, a / 127.0f };
}
// rint(x r) as a byte; a row without a scale (r = 0) stores zeros whatever it holds
__device__ __forceinline__ int k8_code(float x, float r) { return r == 0.0f ? 0 : (int)rintf(x * r); }

template <class T>
__global__ __launch_bounds__(256) void k8_rows_k(int64_t m, int k, const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ q, int64_t ldq, float *__restrict__ s) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= m) return;
    const T *xr = x + row * ldx;
    unsigned top = 0;
    for (int c = lane; c < k; c += 64) top = max(top, k8_mag(k8_f32(xr[c])));
    for (int o = 32; o; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    const RowScale rs = k8_scale(top);
    int8_t *qr = q + row * ldq;
    const int pad = (int)min((int64_t)((k + 15) & ~15), ldq);
    for (int c = lane; c < pad; c += 64) qr[c] = c < k ? (int8_t)k8_code(k8_f32(xr[c]), rs.r) : (int8_t)0;
    if (lane == 0) s[row] = rs.s;
}

template <class T>
__global__ __launch_bounds__(256) void k8_restore_k(int64_t m, int k, const int8_t *__restrict__ q, int64_t ldq, const float *__restrict__ s, T *__restrict__ x, int64_t ldx) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= m) return;
    const float sc = s[row];
    for (int c = threadIdx.x & 63; c < k; c += 64) x[row * ldx + c] = k8_to<T>((float)q[row * ldq + c] * sc);
}

__device__ __forceinline__ bool k8_bit(const uint8_t *mask, int64_t ld, int64_t m, int n) { return !mask || (mask[m * ld + (n >> 3)] >> (n & 7) & 1); }

template <class T>
__global__ __launch_bounds__(256) void k8_linear_k(dn_i8_linear_desc d, const int8_t *__restrict__ q, int64_t ldq, const float *__restrict__ s) {
    const int64_t nb = (d.n + 255) / 256, row = blockIdx.x / nb;
    const int n = (int)(blockIdx.x % nb) * 256 + threadIdx.x;
    float v = 0.0f;
    if (n < d.n) {
        const int8_t *a = q + row * ldq, *b = d.w + (int64_t)n * d.ldw;
        int acc = 0;
        for (int k = 0; k < d.k; k++) acc += (int)a[k] * (int)b[k];
        v = (float)acc * d.sw[n] * s[row];                 // the row's scale last: a row near fp32's end overflows only if its result does
        if (d.bias) v += d.bias[n];
        if (d.residual) v += k8_f32(((const T *)d.residual)[row * d.ldr + n]);
        ((T *)d.y)[row * d.ldy + n] = k8_to<T>(d.relu && v <= 0.0f ? 0.0f : v);
    }
    if (d.mask) {
        const unsigned long long b = __ballot(n < d.n && v > 0.0f);
        if (n < d.n && (threadIdx.x & 7) == 0) d.mask[row * d.ldmask + (n >> 3)] = (uint8_t)(b >> (threadIdx.x & 63));
    }
}

template <class T>
__global__ __launch_bounds__(256) void k8_dx_k(dn_i8_grad_desc d) {
    const int64_t kb = (d.k + 255) / 256, row = blockIdx.x / kb;
    const int k = (int)(blockIdx.x % kb) * 256 + threadIdx.x;
    if (k >= d.k) return;
    float acc = 0.0f;
    for (int n = 0; n < d.n; n++)
        if (k8_bit(d.mask, d.ldmask, row, n)) acc += k8_f32(((const T *)d.dy)[row * d.ldy + n]) * d.sw[n] * (float)d.w[(int64_t)n * d.ldw + k];
    ((T *)d.dx)[row * d.ldx + k] = k8_to<T>(acc);
}

template <class T, class W>
__global__ __launch_bounds__(256) void k8_dw_k(dn_i8_grad_desc d) {
    const int64_t kb = (d.k + 255) / 256;
    const int n = (int)(blockIdx.x / kb), k = (int)(blockIdx.x % kb) * 256 + threadIdx.x;
    float acc = 0.0f, sum = 0.0f;
    for (int64_t m = 0; m < d.m; m++)
        {
            const float g = k8_bit(d.mask, d.ldmask, m, n) ? k8_f32(((const T *)d.dy)[m * d.ldy + n]) : 0.0f;
            sum += g;
            if (k < d.k) acc += g * d.s[m] * (float)d.q[m * d.ldq + k];
        }
    if (d.dw && k < d.k) ((W *)d.dw)[n * d.lddw + k] = k8_to<W>(acc);
    if (d.db && k == 0) ((W *)d.db)[n] = k8_to<W>(sum);
}

constexpr uint64_t k8_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

}  // namespace

#define K8_TYPE(type_, T_, ...) \
    switch (type_) { case DN_T_F32: { typedef float T_; __VA_ARGS__; break; } case DN_T_F16: { typedef _Float16 T_; __VA_ARGS__; break; } \
                     default: { typedef bf16 T_; __VA_ARGS__; break; } }

hipError_t k8_rows(int64_t m, int64_t k, const void *x, int64_t ldx, int x_type, int8_t *q, int64_t ldq, float *s, hipStream_t st) {
    if (m == 0) return hipSuccess;
    K8_TYPE(x_type, T, k8_rows_k<T><<<dim3((unsigned)((m + 3) / 4)), 256, 0, st>>>(m, (int)k, (const T *)x, ldx, q, ldq, s));
    return hipGetLastError();
}

hipError_t k8_restore(int64_t m, int64_t k, const int8_t *q, int64_t ldq, const float *s, void *x, int64_t ldx, int x_type, hipStream_t st) {
    if (m == 0) return hipSuccess;
    K8_TYPE(x_type, T, k8_restore_k<T><<<dim3((unsigned)((m + 3) / 4)), 256, 0, st>>>(m, (int)k, q, ldq, s, (T *)x, ldx));
    return hipGetLastError();
}

// workspace: the rows in 8 bits and their scales, where the caller does not keep them
uint64_t k8_linear_workspace(const dn_i8_linear_desc &d) {
    if (d.x_type == DN_T_I8 || d.q) return 0;
    return k8_up((uint64_t)d.m * k8_up(d.k, 16), 256) + k8_up((uint64_t)d.m * 4, 256);
}

hipError_t k8_linear(const dn_i8_linear_desc &d, void *ws, hipStream_t st) {
    if (d.m == 0) return hipSuccess;
    const int8_t *q = (const int8_t *)d.x; int64_t ldq = d.ldx; const float *s = d.sx;
    if (d.x_type != DN_T_I8) {
        int8_t *qo = d.q; float *so = d.s;
        if (qo) ldq = d.ldq;
        else { ldq = (int64_t)k8_up(d.k, 16); qo = (int8_t *)ws; so = (float *)((char *)ws + k8_up((uint64_t)d.m * ldq, 256)); }
        const hipError_t e = k8_rows(d.m, d.k, d.x, d.ldx, d.x_type, qo, ldq, so, st);
        if (e != hipSuccess) return e;
        q = qo; s = so;
    }
    const unsigned grid = (unsigned)(d.m * ((d.n + 255) / 256));
    K8_TYPE(d.y_type, T, k8_linear_k<T><<<dim3(grid), 256, 0, st>>>(d, q, ldq, s));
    return hipGetLastError();
}

uint64_t k8_grad_workspace(const dn_i8_grad_desc &) { return 0; }

hipError_t k8_grad(const dn_i8_grad_desc &d, void *, hipStream_t st) {
    const int64_t kb = (d.k + 255) / 256;
    K8_TYPE(d.dy_type, T,
            if (d.dx && d.m) k8_dx_k<T><<<dim3((unsigned)(d.m * kb)), 256, 0, st>>>(d);
            if (d.dw || d.db) K8_TYPE(d.dw_type, W, k8_dw_k<T, W><<<dim3((unsigned)(d.n * kb)), 256, 0, st>>>(d)));
    return hipGetLastError();
}
