// k8_grad.hip -- the gradient of the 8-bit dense layers (include/dnascent_hip.h has the formulas).
#include "k8_dense.h"
#include "k8_dev.h"

namespace {

template <class T> __device__ __forceinline__ float k8_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T k8_to(float v) { return (T)v; }
__device__ __forceinline__ bool k8_bit(const uint8_t *mask, int64_t ld, int64_t m, int n) { return !mask || (mask[m * ld + (n >> 3)] >> (n & 7) & 1); }

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

}  // namespace

#define K8_TYPE(type_, T_, ...) \
    switch (type_) { case DN_T_F32: { typedef float T_; __VA_ARGS__; break; } case DN_T_F16: { typedef _Float16 T_; __VA_ARGS__; break; } \
                     default: { typedef k8_bf16 T_; __VA_ARGS__; break; } }

uint64_t k8_grad_workspace(const dn_i8_grad_desc &) { return 0; }

hipError_t k8_grad(const dn_i8_grad_desc &d, void *, hipStream_t st) {
    const int64_t kb = (d.k + 255) / 256;
    K8_TYPE(d.dy_type, T,
            if (d.dx && d.m) k8_dx_k<T><<<dim3((unsigned)(d.m * kb)), 256, 0, st>>>(d);
            if (d.dw || d.db) K8_TYPE(d.dw_type, W, k8_dw_k<T, W><<<dim3((unsigned)(d.n * kb)), 256, 0, st>>>(d)));
    return hipGetLastError();
}
