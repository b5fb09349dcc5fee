// k8_dense.h -- what dn_capi.hip and k8_dense.hip share: the launchers of the 8-bit dense layers.
#pragma once
#include "dnascent_hip.h"
#include <hip/hip_runtime.h>
#include <algorithm>

// every launcher returns hipGetLastError() of its launches; sizes, types and pointers are checked by the C entries
hipError_t k8_rows(int64_t m, int64_t k, const void *x, int64_t ldx, int x_type, int8_t *q, int64_t ldq, float *s, hipStream_t st);
hipError_t k8_restore(int64_t m, int64_t k, const int8_t *q, int64_t ldq, const float *s, void *x, int64_t ldx, int x_type, hipStream_t st);
uint64_t k8_linear_workspace(const dn_i8_linear_desc &d);
hipError_t k8_linear(const dn_i8_linear_desc &d, void *ws, hipStream_t st);
uint64_t k8_grad_workspace(const dn_i8_grad_desc &d);
hipError_t k8_grad(const dn_i8_grad_desc &d, void *ws, hipStream_t st);
