// k8_dense.hip -- 8-bit dense layers: rows in 8 bits and their product (include/dnascent_hip.h has the formulas; the gradient is in k8_grad.hip).
#include "k8_dense.h"
#include "k8_dev.h"

namespace {

// ---- rows in 8 bits ------------------------------------------------------------------------------------------------------------------------------------
// One pass: LPR lanes hold a row in registers (V pieces of 16 bytes each), find the largest magnitude, write the codes.  R rows at a time per lane group
// where a row is one piece per lane, so that enough loads are in flight.  HBM: 2 Mi x 256 bf16, 265 us, 6.1 TB/s; back, 273 us, 5.9 TB/s; 8192 x 4096 bf16, 19 us.
template <class T, int LPR, int V, int R>
__global__ __launch_bounds__(256) void k8_rows_k(int64_t m, int k, const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ q, int64_t ldq, float *__restrict__ s) {
    constexpr int E = 16 / sizeof(T);
    const int lid = threadIdx.x % LPR;
    const int64_t row0 = (int64_t)blockIdx.x * (256 / LPR) * R + threadIdx.x / LPR;      // row i of a lane group: adjacent groups hold adjacent rows
    K8Vec<T, E> raw[R][V];
    unsigned top[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const T *xr = x + min(row0 + i * (256 / LPR), m - 1) * ldx;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int c = (v * LPR + lid) * E;
            if (c + E <= k) raw[i][v] = k8_load<T, E>(xr + c);
            else
#pragma unroll
                for (int e = 0; e < E; e++) raw[i][v].v[e] = c + e < k ? xr[c + e] : (T)0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        top[i] = 0;
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int e = 0; e < E; e++) top[i] = max(top[i], k8_mag((float)raw[i][v].v[e]));
#pragma unroll
        for (int o = (LPR < 64 ? LPR : 64) / 2; o; o >>= 1) top[i] = max(top[i], (unsigned)__shfl_xor((int)top[i], o));
    }
    if (LPR == 256) {
        __shared__ unsigned part[4];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top[0];
        __syncthreads();
        top[0] = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    const int pad = (int)min((int64_t)((k + 15) & ~15), ldq);
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int64_t row = row0 + i * (256 / LPR);
        if (row >= m) break;
        const K8Scale sc = k8_scale(top[i]);
        int8_t *qr = q + row * ldq;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int c = (v * LPR + lid) * E;
            K8Vec<unsigned, E / 4> w;
#pragma unroll
            for (int e = 0; e < E / 4; e++)
                w.v[e] = k8_codes((float)raw[i][v].v[4 * e], (float)raw[i][v].v[4 * e + 1], (float)raw[i][v].v[4 * e + 2], (float)raw[i][v].v[4 * e + 3], sc.r);
            if (c + E <= pad) __builtin_memcpy(qr + c, &w, E);
            else
#pragma unroll
                for (int e = 0; e < E; e++) if (c + e < pad) qr[c + e] = (int8_t)(w.v[e / 4] >> (8 * (e % 4)));
        }
        if (lid == 0) s[row] = sc.s;
    }
}
// rows that do not fit a workgroup's registers: read twice (the second time mostly from cache)
template <class T>
__global__ __launch_bounds__(256) void k8_rows_long(int k, const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ q, int64_t ldq, float *__restrict__ s) {
    constexpr int E = 16 / sizeof(T);
    const T *xr = x + (int64_t)blockIdx.x * ldx;
    int8_t *qr = q + (int64_t)blockIdx.x * ldq;
    const int whole = k / E * E;
    unsigned top = 0;
#pragma unroll 4
    for (int c = threadIdx.x * E; c < whole; c += 256 * E) {
        const K8Vec<T, E> r = k8_load<T, E>(xr + c);
#pragma unroll
        for (int e = 0; e < E; e++) top = max(top, k8_mag((float)r.v[e]));
    }
    if (whole + (int)threadIdx.x < k) top = max(top, k8_mag((float)xr[whole + threadIdx.x]));
    for (int o = 32; o; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    __shared__ unsigned part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    const K8Scale sc = k8_scale(max(max(part[0], part[1]), max(part[2], part[3])));
#pragma unroll 4
    for (int c = threadIdx.x * E; c < whole; c += 256 * E) {
        const K8Vec<T, E> r = k8_load<T, E>(xr + c);
        K8Vec<unsigned, E / 4> w;
#pragma unroll
        for (int e = 0; e < E / 4; e++) w.v[e] = k8_codes((float)r.v[4 * e], (float)r.v[4 * e + 1], (float)r.v[4 * e + 2], (float)r.v[4 * e + 3], sc.r);
        __builtin_memcpy(qr + c, &w, E);
    }
    const int c = whole + threadIdx.x, pad = (int)min((int64_t)((k + 15) & ~15), ldq);
    if (c < pad) qr[c] = c < k && sc.r != 0.0f ? (int8_t)k8_code((float)xr[c], sc.r) : (int8_t)0;
    if (threadIdx.x == 0) s[blockIdx.x] = sc.s;
}

template <class T>
hipError_t rows_of(int64_t m, int k, const T *x, int64_t ldx, int8_t *q, int64_t ldq, float *s, hipStream_t st) {
    constexpr int E = 16 / sizeof(T);
#define ROWS(LPR_, V_, R_) k8_rows_k<T, LPR_, V_, R_><<<dim3((unsigned)((m + (256 / LPR_) * R_ - 1) / ((256 / LPR_) * R_))), 256, 0, st>>>(m, k, x, ldx, q, ldq, s)
    // a wavefront or less per row up to 128 pieces of 16 bytes, if there are rows enough to fill the chip that way; a workgroup per row for few or long rows.  Rows and back,
    // bf16, us, wavefront : workgroup -- 200000 x 1000, 224 : 304; 100000 x 600, 67 : 119; 100 x 1000, 7.1 : 5.7; 8192 x 4096, 37 : 33; 2048 x 4096, 11.9 : 10.5
    const int pieces = (k + E - 1) / E;
    if (pieces <= 8) ROWS(8, 1, 4);
    else if (pieces <= 16) ROWS(16, 1, 4);
    else if (pieces <= 32) ROWS(32, 1, 4);
    else if (pieces <= 64) ROWS(64, 1, 4);
    else if (pieces <= 128 && m >= 8 * K8_CUS) ROWS(64, 2, 2);
    else if (pieces <= 256) ROWS(256, 1, 1);
    else if (pieces <= 512) ROWS(256, 2, 1);
    else if (pieces <= 1024) ROWS(256, 4, 1);
    else if (pieces <= 2048) ROWS(256, 8, 1);
    else k8_rows_long<T><<<dim3((unsigned)m), 256, 0, st>>>(k, x, ldx, q, ldq, s);
#undef ROWS
    return hipGetLastError();
}

template <class T, int LPR, int R>
__global__ __launch_bounds__(256) void k8_restore_k(int64_t m, int k, const int8_t *__restrict__ q, int64_t ldq, const float *__restrict__ s, T *__restrict__ x, int64_t ldx) {
    constexpr int E = 16 / sizeof(T);
    const int lid = threadIdx.x % LPR;
    const int64_t row0 = (int64_t)blockIdx.x * (256 / LPR) * R + threadIdx.x / LPR;
    for (int c = lid * E; c < k; c += LPR * E) {
        K8Vec<int8_t, E> raw[R];
        float sc[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int64_t row = min(row0 + i * (256 / LPR), m - 1);
            sc[i] = s[row];
            if (c + E <= k) raw[i] = k8_load<int8_t, E>(q + row * ldq + c);
            else
#pragma unroll
                for (int e = 0; e < E; e++) raw[i].v[e] = c + e < k ? q[row * ldq + c + e] : (int8_t)0;
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int64_t row = row0 + i * (256 / LPR);
            if (row >= m) break;
            T *xr = x + row * ldx + c;
            K8Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; e++) o.v[e] = (T)((float)raw[i].v[e] * sc[i]);
            if (c + E <= k) k8_stream<T, E>(xr, o);
            else
#pragma unroll
                for (int e = 0; e < E; e++) if (c + e < k) xr[e] = o.v[e];
        }
    }
}
template <class T>
hipError_t restore_of(int64_t m, int k, const int8_t *q, int64_t ldq, const float *s, T *x, int64_t ldx, hipStream_t st) {
    const int pieces = (int)((k + 16 / sizeof(T) - 1) / (16 / sizeof(T)));
#define REST(LPR_, R_) k8_restore_k<T, LPR_, R_><<<dim3((unsigned)((m + (256 / LPR_) * R_ - 1) / ((256 / LPR_) * R_))), 256, 0, st>>>(m, k, q, ldq, s, x, ldx)
    if (pieces <= 8) REST(8, 4);
    else if (pieces <= 16) REST(16, 4);
    else if (pieces <= 32) REST(32, 4);
    else if (pieces <= 64 && m >= 8 * K8_CUS) REST(64, 4);
    else if (pieces <= 128 && m >= 8 * K8_CUS) REST(64, 1);
    else REST(256, 1);
#undef REST
    return hipGetLastError();
}

// ---- what happens to a sum ---------------------------------------------------------------------------------------------------------------------------------
struct Out {                                               // the epilogue's half of dn_i8_linear_desc
    const float *sx, *sw, *bias; const void *residual; void *y; uint8_t *mask;
    int64_t m, n, ldr, ldy, ldmask; int relu;
};
__device__ __forceinline__ float k8_finish(int acc, float sw, float sx, float bias) {
    return (float)acc * sw * sx + bias;                    // the row's scale last: a row near fp32's end overflows only if its result does
}
// TN adjacent columns of one row: what is added to them, and where they go
template <class T, int TN>
__device__ __forceinline__ K8Vec<T, TN> k8_added(const Out &o, int64_t mm, int64_t nn) {
    K8Vec<T, TN> t;
    const T *r = (const T *)o.residual + mm * o.ldr + nn;
    if (nn + TN <= o.n) t = k8_load<T, TN>(r);
    else
#pragma unroll
        for (int j = 0; j < TN; j++) t.v[j] = nn + j < o.n ? r[j] : (T)0.0f;
    return t;
}
template <class T, int TN>
__device__ __forceinline__ void k8_put(const Out &o, int64_t mm, int64_t nn, const float (&v)[TN]) {
    K8Vec<T, TN> y;
#pragma unroll
    for (int j = 0; j < TN; j++) y.v[j] = (T)(o.relu ? k8_relu(v[j]) : v[j]);
    T *p = (T *)o.y + mm * o.ldy + nn;
    if (nn + TN <= o.n) k8_stream<T, TN>(p, y);
    else
#pragma unroll
        for (int j = 0; j < TN; j++) if (nn + j < o.n) p[j] = y.v[j];
}
// The mask's bits: the 32 lanes of a half wavefront hold 32 TN adjacent columns of a row; lanes put their TN bits together into bytes (the columns of a half start
// at a multiple of 32 TN, so bytes never straddle halves)
template <int TN>
__device__ __forceinline__ void k8_put_mask(const Out &o, int64_t mm, int64_t nn, const float (&v)[TN], bool live) {
    // every lane of the wavefront comes here; 8 / TN neighbouring lanes share a byte
    unsigned b = 0;
#pragma unroll
    for (int j = 0; j < TN; j++) b |= (live && nn + j < o.n && v[j] > 0.0f ? 1u : 0u) << j;
    b <<= ((unsigned)nn & 7u);
#pragma unroll
    for (int q = 1; q < 8 / TN; q <<= 1) b |= (unsigned)__shfl_xor((int)b, q);
    if (live && (nn & 7) == 0) o.mask[mm * o.ldmask + (nn >> 3)] = (uint8_t)b;
}

template <class T>
struct LinearEpi {
    typedef int value;
    Out o;
    template <int TN> struct Columns { float sw[TN], bias[TN]; };
    template <int TN> __device__ __forceinline__ Columns<TN> columns(int64_t nn) const {
        Columns<TN> c;
#pragma unroll
        for (int j = 0; j < TN; j++) { const int64_t n = min(nn + j, o.n - 1); c.sw[j] = o.sw[n]; c.bias[j] = o.bias ? o.bias[n] : 0.0f; }
        return c;
    }
    template <int TN> struct Row { float sx; K8Vec<T, TN> added; };
    template <int TN> __device__ __forceinline__ Row<TN> row(int64_t mm, int64_t nn) const {
        Row<TN> r;
        r.sx = o.sx[mm];
        if (o.residual) r.added = k8_added<T, TN>(o, mm, nn);
        return r;
    }
    template <int TN> __device__ __forceinline__ void store(const Columns<TN> &c, const Row<TN> &r, int64_t mm, int64_t nn, int, const int (&acc)[TN], bool live) const {
        float v[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) v[j] = k8_finish(acc[j], c.sw[j], r.sx, c.bias[j]);
        if (o.residual)
#pragma unroll
            for (int j = 0; j < TN; j++) v[j] += (float)r.added.v[j];
        if (live) k8_put<T, TN>(o, mm, nn, v);
        if (o.mask) k8_put_mask<TN>(o, mm, nn, v, live);
    }
};
// a run's sums as they are: part [splits][m][n]
struct PartEpi {
    typedef int value;
    int *part; int64_t m, n;
    template <int TN> struct Columns {};
    template <int TN> __device__ __forceinline__ Columns<TN> columns(int64_t) const { return {}; }
    template <int TN> struct Row {};
    template <int TN> __device__ __forceinline__ Row<TN> row(int64_t, int64_t) const { return {}; }
    template <int TN> __device__ __forceinline__ void store(const Columns<TN> &, const Row<TN> &, int64_t mm, int64_t nn, int z, const int (&acc)[TN], bool live) const {
        if (!live) return;
        int *p = part + ((int64_t)z * m + mm) * n + nn;
        K8Vec<int, TN> v;
#pragma unroll
        for (int j = 0; j < TN; j++) v.v[j] = acc[j];
        if (nn + TN <= n) k8_store<int, TN>(p, v);
        else
#pragma unroll
            for (int j = 0; j < TN; j++) if (nn + j < n) p[j] = acc[j];
    }
};
// the runs joined: a wavefront takes 256 adjacent columns of a row, four per lane
template <class T>
__global__ __launch_bounds__(256) void k8_join(const int *__restrict__ part, int splits, Out o) {
    const int64_t nb = (o.n + 255) / 256, w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= o.m * nb) return;
    const int64_t mm = w / nb, nn = (w % nb) * 256 + (threadIdx.x & 63) * 4;
    const bool live = nn < o.n;
    int acc[4] = { 0, 0, 0, 0 };
    if (live)
#pragma unroll 4
        for (int z = 0; z < splits; z++) {
            const int *p = part + ((int64_t)z * o.m + mm) * o.n + nn;
            if (nn + 4 <= o.n) {
                const K8Vec<int, 4> t = k8_load<int, 4>(p);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[j] += t.v[j];
            } else
#pragma unroll
                for (int j = 0; j < 4; j++) if (nn + j < o.n) acc[j] += p[j];
        }
    const LinearEpi<T> e{ o };
    e.template store<4>(e.template columns<4>(live ? nn : 0), e.template row<4>(mm, live ? nn : 0), mm, nn, 0, acc, live);
}

// rows at a pitch the product cannot fetch (not a multiple of 16 bytes), copied to one that it can, zeros behind their ends
__global__ __launch_bounds__(256) void k8_repitch(const int8_t *__restrict__ src, int64_t ld, int64_t rows, int k, int8_t *__restrict__ dst, int pitch) {
    const int64_t total = rows * (pitch / 16), step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const int64_t r = i / (pitch / 16);
        const int c = (int)(i - r * (pitch / 16)) * 16;
        K8Vec<int8_t, 16> v;
        if (c + 16 <= k) v = k8_load<int8_t, 16>(src + r * ld + c);
        else
#pragma unroll
            for (int e = 0; e < 16; e++) v.v[e] = c + e < k ? src[r * ld + c + e] : (int8_t)0;
        *(i32x4 *)(dst + r * pitch + c) = __builtin_bit_cast(i32x4, v);
    }
}

// ---- few rows (M <= 64): the weight is streamed once ---------------------------------------------------------------------------------------------------------
// A workgroup takes 16 output channels; its eight wavefronts cut K into steps of 64 and join their sums in LDS.  The weight goes straight from memory into
// the matrix instructions' operands, eight steps in flight per wavefront.  Rows that arrive as numbers are put into 8 bits by every workgroup for itself
// (X != int8_t: they are few, and a second launch costs more than reading them again from L2).  Bound by the latency from the first load to the last store:
// 1 x 4096 x 4096 bf16 7.2 us (16.8 MB, 2.3 TB/s), 1 x 256 x 256 6.0 us, 13 given rows x 4352 x 1000 6.0 us.
template <class X, int MT>
__global__ __launch_bounds__(512) void k8_few(const X *__restrict__ x, int64_t ldx, const int8_t *__restrict__ w, int64_t ldw, int k, Out o, int y_type,
                                              int8_t *__restrict__ qout, int64_t ldq, float *__restrict__ sout) {
    extern __shared__ __align__(16) char dyn[];            // X != int8_t: the rows' codes at a pitch of kp + 16 bytes
    __shared__ int sums[8][MT * 256];
    __shared__ float scales[MT * 16];
    __shared__ unsigned tops[8];
    constexpr bool GIVEN = sizeof(X) == 1;
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4, m = (int)o.m;
    const int kp = (k + 63) & ~63, pitch = kp + 16, mine = min(c, m - 1);      // operand rows behind the last one repeat it
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int steps = kp >> 6, whole = k >> 6;             // whole: steps that no lane has to cut
    const int8_t *wr = w + min(n0 + c, o.n - 1) * ldw;
    // the first eight steps of the weight are asked for before anything else
    i32x4 b[8];
    const bool eight = wave + 56 < whole;
    if (eight)
#pragma unroll
        for (int u = 0; u < 8; u++) b[u] = __builtin_bit_cast(i32x4, k8_load<int8_t, 16>(wr + (wave + 8 * u) * 64 + g * 16));
    if constexpr (GIVEN) {
        if (threadIdx.x < MT * 16) scales[threadIdx.x] = o.sx[min((int)threadIdx.x, m - 1)];
    } else {
        // 8, 4, 2 or 1 wavefronts a row; M K <= 16384, so that a lane holds its share of a row in eight pieces of eight numbers at most
        const int per = m == 1 ? 8 : m == 2 ? 4 : m <= 4 ? 2 : 1, part = wave % per;
        for (int r = wave / per; r < (m + 8 / per - 1) / (8 / per) * (8 / per); r += 8 / per) {      // (as many rounds for every wavefront)
            const X *xr = x + min(r, m - 1) * ldx;
            K8Raw<X, 8> raw[8];
            unsigned top = 0;
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const int at = ((v * per + part) * 64 + lane) * 8;
                if (at + 8 <= k) raw[v].load(xr + at);
                else if (v * per * 512 < k) raw[v].load(xr + at, k - at);
                else raw[v] = {};
            }
#pragma unroll
            for (int v = 0; v < 8; v++)
#pragma unroll
                for (int e = 0; e < 8; e++) top = max(top, k8_mag(raw[v].get(e)));
            for (int d = 32; d; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
            if (per > 1) {
                if (lane == 0) tops[wave] = top;
                __syncthreads();
                for (int z = 0; z < per; z++) top = max(top, tops[wave / per * per + z]);
            }
            if (r >= m) break;                             // (only where a wavefront has a row to itself: no barrier follows)
            const K8Scale sc = k8_scale(top);
            const int pad = (int)min((int64_t)((k + 15) & ~15), ldq);
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const int at = ((v * per + part) * 64 + lane) * 8;
                if (at >= kp) break;
                const unsigned q0 = k8_codes(raw[v].get(0), raw[v].get(1), raw[v].get(2), raw[v].get(3), sc.r);
                const unsigned q1 = k8_codes(raw[v].get(4), raw[v].get(5), raw[v].get(6), raw[v].get(7), sc.r);
                *(uint2 *)(dyn + r * pitch + at) = make_uint2(q0, q1);
                if (qout && blockIdx.x == 0) {
                    if (at + 8 <= pad) { const uint2 q = make_uint2(q0, q1); __builtin_memcpy(qout + r * ldq + at, &q, 8); }
                    else
#pragma unroll
                        for (int e = 0; e < 8; e++) if (at + e < pad) qout[r * ldq + at + e] = (int8_t)((e < 4 ? q0 : q1) >> (8 * (e & 3)));
                }
            }
            if (lane == 0 && part == 0) { scales[r] = sc.s; if (sout && blockIdx.x == 0) sout[r] = sc.s; }
        }
        __syncthreads();
    }
    i32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] = i32x4{ 0, 0, 0, 0 };
    const int8_t *xr[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) xr[t] = GIVEN ? (const int8_t *)x + min(t * 16 + c, m - 1) * ldx : nullptr;
    auto piece = [&](const int8_t *row, int at) -> i32x4 { // 16 codes of a row, zeros behind its end
        if (at + 16 <= k) return __builtin_bit_cast(i32x4, k8_load<int8_t, 16>(row + at));
        K8Vec<int8_t, 16> v;
#pragma unroll
        for (int e = 0; e < 16; e++) v.v[e] = at + e < k ? row[at + e] : (int8_t)0;
        return __builtin_bit_cast(i32x4, v);
    };
    int s = wave;
    for (; s + 56 < whole; s += 64) {
        if (s != wave)
#pragma unroll
        for (int u = 0; u < 8; u++) b[u] = __builtin_bit_cast(i32x4, k8_load<int8_t, 16>(wr + (s + 8 * u) * 64 + g * 16));
#pragma unroll
        for (int u = 0; u < 8; u++)
#pragma unroll
            for (int t = 0; t < MT; t++) {
                const int at = (s + 8 * u) * 64 + g * 16;
                const i32x4 a = GIVEN ? __builtin_bit_cast(i32x4, k8_load<int8_t, 16>(xr[t] + at)) : *(const i32x4 *)(dyn + mine * pitch + at);
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b[u], acc[t], 0, 0, 0);
            }
    }
    for (; s < steps; s += 8) {
        const int at = s * 64 + g * 16;
        const i32x4 bp = piece(wr, at);
#pragma unroll
        for (int t = 0; t < MT; t++) {
            i32x4 a;
            if constexpr (GIVEN) a = piece(xr[t], at); else a = *(const i32x4 *)(dyn + mine * pitch + at);
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, bp, acc[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; t++)                           // D: column lane & 15, row 4 (lane >> 4) + i
#pragma unroll
        for (int i = 0; i < 4; i++) sums[wave][t * 256 + (4 * g + i) * 16 + c] = acc[t][i];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 256; i += 512) {    // 64 lanes: four rows of 16 columns
        int a = 0;
#pragma unroll
        for (int z = 0; z < 8; z++) a += sums[z][i];
        const int r = i >> 4;
        const int64_t nn = n0 + (i & 15), nc = min(nn, o.n - 1);
        const bool live = r < m && nn < o.n;
        float v[1] = { k8_finish(a, o.sw[nc], scales[min(r, m - 1)], o.bias ? o.bias[nc] : 0.0f) };
        auto put = [&](auto one) __attribute__((always_inline)) {
            typedef decltype(one) Y;
            if (o.residual) v[0] += (float)k8_added<Y, 1>(o, r, nn).v[0];
            k8_put<Y, 1>(o, r, nn, v);
        };
        if (live) {
            if (y_type == DN_T_F32) put(0.0f);
            else if (y_type == DN_T_F16) put((_Float16)0.0f);
            else put((k8_bf16)0.0f);
        }
        if (o.mask) k8_put_mask<1>(o, r, nn, v, live);
    }
}

// ---- many narrow rows (K <= 256): the weight stays in LDS, a row is read once and never leaves the registers as numbers ----------------------------------------
// A wavefront takes 16 rows at a time: a lane holds 16 KS numbers of one row (KS = steps of 64), four lanes a row; they find the row's scale, make the codes --
// which then ARE the matrix instructions' operand -- and multiply them with the weight, whose fragments lie in LDS in the order they are read.  The order of k
// inside a step is free as long as both operands agree: it follows the loads (each lane 16 bytes, a row's four lanes side by side).
// Column tile t of a block of 64 holds columns 4 c + t, so that a lane ends up with four adjacent columns of four rows.
// The next 16 rows are fetched before the products of these.  HBM: 1 Mi x 256 x 256 fp32 with ReLU 415 us, 5.2 TB/s, a copy's rate.
template <class X> constexpr int k8_piece_of(int ks, int g, int b) {                     // which k byte b of lane group g's operand is
    return sizeof(X) == 4 ? ks * 64 + 16 * (b >> 2) + 4 * g + (b & 3) : sizeof(X) == 2 ? ks * 64 + 32 * (b >> 3) + 8 * g + (b & 7) : ks * 64 + 16 * g + b;
}
template <class X, class Y, int KS>
__global__ __launch_bounds__(512) void k8_narrow(const X *__restrict__ x, int64_t ldx, const int8_t *__restrict__ w, int64_t ldw, int k, Out o,
                                                 int8_t *__restrict__ qout, int64_t ldq, float *__restrict__ sout) {
    constexpr int E = 16 / sizeof(X), P = 16 / E;           // numbers per load, loads per step
    constexpr bool GIVEN = sizeof(X) == 1;
    __shared__ __align__(16) char lw[256 * KS * 64];
    __shared__ float lsw[256], lbias[256];
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.y * 256;
    const int cols = (int)min((int64_t)256, o.n - n0), blocks = (cols + 63) / 64;
#pragma unroll 4
    for (int f = threadIdx.x; f < blocks * 4 * KS * 64; f += 512) {
        const int fl = f & 63, ks = (f >> 6) % KS, t = (f >> 6) / KS % 4, blk = (f >> 6) / (KS * 4);
        const int col = blk * 64 + 4 * (fl & 15) + t;
        const int8_t *wr = w + (n0 + min(col, cols - 1)) * ldw;
        // runs of C codes; one that ends behind the row is read in front of its end and moved down.  No branch around a load: it would be waited for there
        constexpr int C = E < 8 ? E : 8;
        uint64_t v[16 / C];
#pragma unroll
        for (int j = 0; j < 16 / C; j++) {
            const int at = k8_piece_of<X>(ks, fl >> 4, j * C), from = min(at, k - C);
            v[j] = 0;
            if (k >= C) __builtin_memcpy(&v[j], wr + from, C);
            else
#pragma unroll
                for (int b = 0; b < C; b++) v[j] |= (uint64_t)(uint8_t)wr[min(b, k - 1)] << (8 * b);
        }
        i32x4 out;
#pragma unroll
        for (int j = 0; j < 16 / C; j++) {
            const int at = k8_piece_of<X>(ks, fl >> 4, j * C), skip = k >= C ? min(max(at + C - k, 0), C) : 0, have = k >= C ? C : max(k - at, 0);
            uint64_t r = skip < 8 ? v[j] >> (8 * skip) : 0;
            if (have < C) r &= (1ull << (8 * have)) - 1;
            out[j * C / 4] = (int)(unsigned)r;
            if (C == 8) out[(j * C / 4 + 1) & 3] = (int)(unsigned)(r >> 32);
        }
        *(i32x4 *)(lw + f * 16) = out;
    }
    for (int i = threadIdx.x; i < 256; i += 512) {
        lsw[i] = i < cols ? o.sw[n0 + i] : 0.0f;
        lbias[i] = i < cols && o.bias ? o.bias[n0 + i] : 0.0f;
    }
    __syncthreads();
    const bool whole = k == KS * 64;
    const int64_t tiles = (o.m + 15) / 16, stride = (int64_t)gridDim.x * 8;
    K8Vec<X, E> raw[KS][P];
    float sx = 0.0f;
    auto fetch = [&](int64_t tile) {
        const int64_t row = min(tile * 16 + c, o.m - 1);
        const X *xr = x + row * ldx;
        if (GIVEN) sx = o.sx[row];
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int p = 0; p < P; p++) {
                const int at = k8_piece_of<X>(ks, g, p * E);
                if (whole || at + E <= k) raw[ks][p] = k8_load<X, E>(xr + at);
                else
#pragma unroll
                    for (int e = 0; e < E; e++) raw[ks][p].v[e] = at + e < k ? xr[at + e] : (X)0;
            }
    };
    int64_t tile = (int64_t)blockIdx.x * 8 + wave;
    if (tile < tiles) fetch(tile);
    for (; tile < tiles; tile += stride) {
        i32x4 a[KS];
        float s;
        if constexpr (GIVEN) {
            s = sx;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) a[ks] = __builtin_bit_cast(i32x4, raw[ks][0]);
        } else {
            unsigned top = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int e = 0; e < E; e++) top = max(top, k8_mag((float)raw[ks][p].v[e]));
            top = max(top, (unsigned)__shfl_xor((int)top, 16));
            top = max(top, (unsigned)__shfl_xor((int)top, 32));
            const K8Scale sc = k8_scale(top);
            s = sc.s;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const K8Vec<X, E> &r = raw[ks][d * 4 / E];
                    const int e = d * 4 % E;
                    a[ks][d] = (int)k8_codes((float)r.v[e], (float)r.v[e + 1], (float)r.v[e + 2], (float)r.v[e + 3], sc.r);
                }
            if (qout && blockIdx.y == 0 && tile * 16 + c < o.m) {
                const int pad = (int)min((int64_t)((k + 15) & ~15), ldq);
                int8_t *qr = qout + (tile * 16 + c) * ldq;
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        const int at = k8_piece_of<X>(ks, g, p * E);
                        if (at + E <= pad) __builtin_memcpy(qr + at, (const char *)&a[ks] + p * E, E);
                        else
#pragma unroll
                            for (int e = 0; e < E; e++) if (at + e < pad) qr[at + e] = ((const int8_t *)&a[ks])[p * E + e];
                    }
                if (g == 0) sout[tile * 16 + c] = s;
            }
        }
        if (tile + stride < tiles) fetch(tile + stride);
        float rs[4];
#pragma unroll
        for (int i = 0; i < 4; i++) rs[i] = __shfl(s, 4 * g + i);
        for (int blk = 0; blk < blocks; blk++) {
            i32x4 acc[4];
            const char *lb = lw + (blk * 4 * KS * 64 + lane) * 16;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                acc[t] = i32x4{ 0, 0, 0, 0 };
#pragma unroll
                for (int ks = 0; ks < KS; ks++) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[ks], *(const i32x4 *)(lb + (t * KS + ks) * 1024), acc[t], 0, 0, 0);
            }
            const k8_f32x4 sw = *(const k8_f32x4 *)(lsw + blk * 64 + 4 * c), bias = *(const k8_f32x4 *)(lbias + blk * 64 + 4 * c);
            const int64_t nn = n0 + blk * 64 + 4 * c;
            K8Vec<Y, 4> added[4];
            if (o.residual)
#pragma unroll
                for (int i = 0; i < 4; i++) added[i] = k8_added<Y, 4>(o, min(tile * 16 + 4 * g + i, o.m - 1), nn);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t mm = tile * 16 + 4 * g + i;
                float v[4];
#pragma unroll
                for (int t = 0; t < 4; t++) v[t] = k8_finish(acc[t][i], sw[t], rs[i], bias[t]);
                if (o.residual)
#pragma unroll
                    for (int t = 0; t < 4; t++) v[t] += (float)added[i].v[t];
                const bool live = mm < o.m && nn < o.n;
                if (live) k8_put<Y, 4>(o, mm, nn, v);
                if (o.mask) k8_put_mask<4>(o, mm, nn, v, live);
            }
        }
    }
}

// ---- which way a call takes ---------------------------------------------------------------------------------------------------------------------------------
enum { FEW, NARROW, WIDE };
struct Plan {
    int way = WIDE, splits = 1; K8Tiling tile = K8_BIG; bool inside = false;
    uint64_t q = 0, s = 0, x = 0, w = 0, part = 0, total = 0;   // places in the workspace
    int64_t ldq = 0;
};
inline bool k8_direct(const void *p, int64_t ld) { return ((uintptr_t)p | (uint64_t)ld) % 16 == 0; }
Plan plan_linear(const dn_i8_linear_desc &d) {
    Plan p;
    const bool given = d.x_type == DN_T_I8;
    auto take = [&](uint64_t bytes) { const uint64_t at = p.total; p.total += k8_up(bytes, 256); return at; };
    // few rows: one launch (or two) without tiles of 128 rows.  us, this : tiles, bf16, 4096 x 4096 -- 17 rows, 10 : 15; 64 rows, 16 : 17; 64 x 1000 x 1000, 11 : 13
    if (d.m <= 64) p.way = FEW;
    // Narrow rows: one launch that reads x once, but every workgroup first lays out its 256 channels of the weight (K > 128: 10 us).  us, this : rows and tiles, bf16 --
    // 200 x 64 x 64, 5.7 : 9.8; 100000 x 64 x 512, 41 : 73; 20000 x 128 x 2048, 47 : 56; 5000 x 256 x 256, 17 : 12; 50000 x 256 x 256, 34 : 35; 1048576 x 256 x 256, 383 : 475;
    // 20000 x 256 x 512, 35 : 29; 20000 x 256 x 1024, 42 : 46
    else if ((given || d.x_type == d.y_type) && (d.k <= 128 ? d.n <= 2048 : d.k <= 256 && d.n <= 1024 && d.m * ((d.n + 255) / 256) >= 49152)) { p.way = NARROW; return p; }
    // few rows of numbers: their codes fit a workgroup's LDS beside its sums.  That saves a launch and a workspace (3 us of a call); on the device alone it costs as much
    // (1 x 4096 x 4096: 8.3 us, in two launches 8.1; 16 x 1024 x 1024: 8.8 and 6.5)
    p.inside = p.way == FEW && !given && d.m <= 16 && d.m * d.k <= 16384;
    if (p.inside) return p;
    if (!given && !d.q) {
        p.ldq = (int64_t)k8_up(d.k, 16);
        p.q = take((uint64_t)d.m * p.ldq); p.s = take((uint64_t)d.m * 4);
    }
    if (p.way == FEW) return p;
    if (given ? !k8_direct(d.x, d.ldx) : d.q && !k8_direct(d.q, d.ldq)) p.x = take((uint64_t)d.m * k8_up(d.k, 16));
    if (!k8_direct(d.w, d.ldw)) p.w = take((uint64_t)d.n * k8_up(d.k, 16));
    p.tile = k8_tiling(d.m, d.n);
    const int64_t tiles = k8_tiles(p.tile, d.m, d.n);
    if (tiles < K8_CUS) {                                  // fewer tiles than compute units: the reduction is cut, four steps at least to a run
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(K8_CUS / tiles, ((d.k + 127) / 128) / 4));
        if (p.splits > 1) p.part = take((uint64_t)p.splits * d.m * d.n * 4);
    }
    return p;
}

}  // namespace

#define K8_TYPE(type_, T_, ...) \
    switch (type_) { case DN_T_F32: { typedef float T_; __VA_ARGS__; break; } case DN_T_F16: { typedef _Float16 T_; __VA_ARGS__; break; } \
                     default: { typedef k8_bf16 T_; __VA_ARGS__; break; } }

hipError_t k8_rows(int64_t m, int64_t k, const void *x, int64_t ldx, int x_type, int8_t *q, int64_t ldq, float *s, hipStream_t st) {
    for (int64_t r = 0; r < m; r += K8_LAUNCH_ROWS) {
        hipError_t e = hipSuccess;
        K8_TYPE(x_type, T, e = rows_of<T>(std::min(m - r, K8_LAUNCH_ROWS), (int)k, (const T *)x + r * ldx, ldx, q + r * ldq, ldq, s + r, st));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t k8_restore(int64_t m, int64_t k, const int8_t *q, int64_t ldq, const float *s, void *x, int64_t ldx, int x_type, hipStream_t st) {
    for (int64_t r = 0; r < m; r += K8_LAUNCH_ROWS) {
        hipError_t e = hipSuccess;
        K8_TYPE(x_type, T, e = restore_of<T>(std::min(m - r, K8_LAUNCH_ROWS), (int)k, q + r * ldq, ldq, s + r, (T *)x + r * ldx, ldx, st));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

uint64_t k8_linear_workspace(const dn_i8_linear_desc &d) { return plan_linear(d).total; }

hipError_t k8_linear(const dn_i8_linear_desc &d, void *ws, hipStream_t st) {
    if (d.m == 0) return hipSuccess;
    const Plan p = plan_linear(d);
    char *base = (char *)ws;
    const bool given = d.x_type == DN_T_I8;
    Out o = { d.sx, d.sw, d.bias, d.residual, d.y, d.mask, d.m, d.n, d.ldr, d.ldy, d.ldmask, d.relu };
    if (p.way == NARROW) {
        const unsigned per = (unsigned)((d.n + 255) / 256), wgs = (unsigned)std::min<int64_t>((d.m + 127) / 128, 2 * K8_CUS / per);
        const int steps = (int)((d.k + 63) / 64);
#define NARROW_GO(X_, Y_, KS_) k8_narrow<X_, Y_, KS_><<<dim3(wgs, per), 512, 0, st>>>((const X_ *)d.x, d.ldx, d.w, d.ldw, (int)d.k, o, d.q, d.ldq, d.s)
#define NARROW_KS(X_, Y_) do { if (steps == 1) NARROW_GO(X_, Y_, 1); else if (steps == 2) NARROW_GO(X_, Y_, 2); else NARROW_GO(X_, Y_, 4); } while (0)
        if (given) { K8_TYPE(d.y_type, T, NARROW_KS(int8_t, T)); } else { K8_TYPE(d.y_type, T, NARROW_KS(T, T)); }
#undef NARROW_KS
#undef NARROW_GO
        return hipGetLastError();
    }
    const unsigned few_grid = (unsigned)((d.n + 15) / 16);
    if (p.inside) {
        const unsigned lds = (unsigned)(d.m * (k8_up(d.k, 64) + 16));
        K8_TYPE(d.x_type, T, k8_few<T, 1><<<dim3(few_grid), 512, lds, st>>>((const T *)d.x, d.ldx, d.w, d.ldw, (int)d.k, o, d.y_type, d.q, d.ldq, d.s));
        return hipGetLastError();
    }
    const int8_t *q = (const int8_t *)d.x; int64_t ldq = d.ldx;
    if (!given) {
        int8_t *qo = d.q ? d.q : (int8_t *)(base + p.q); float *so = d.q ? d.s : (float *)(base + p.s);
        ldq = d.q ? d.ldq : p.ldq;
        const hipError_t e = k8_rows(d.m, d.k, d.x, d.ldx, d.x_type, qo, ldq, so, st);
        if (e != hipSuccess) return e;
        q = qo; o.sx = so;
    }
    if (p.way == FEW) {
#define FEW_GO(MT_) k8_few<int8_t, MT_><<<dim3(few_grid), 512, 0, st>>>(q, ldq, d.w, d.ldw, (int)d.k, o, d.y_type, nullptr, 0, nullptr)
        if (d.m <= 16) FEW_GO(1); else if (d.m <= 32) FEW_GO(2); else FEW_GO(4);
#undef FEW_GO
        return hipGetLastError();
    }
    const int8_t *w = d.w; int64_t ldw = d.ldw;
    const int pitch = (int)k8_up(d.k, 16);
    auto repitch = [&](const int8_t *src, int64_t ld, int64_t rows, uint64_t at) {
        k8_repitch<<<dim3((unsigned)std::min<int64_t>((rows * (pitch / 16) + 255) / 256, 8 * K8_CUS)), 256, 0, st>>>(src, ld, rows, (int)d.k, (int8_t *)base + at, pitch);
        return (const int8_t *)base + at;
    };
    if (!k8_direct(q, ldq)) { q = repitch(q, ldq, d.m, p.x); ldq = pitch; }
    if (!k8_direct(w, ldw)) { w = repitch(w, ldw, d.n, p.w); ldw = pitch; }
    G8 g = { (const char *)q, (const char *)w, ldq, ldw, d.m, d.n, (int)d.k, 1, 0, p.splits, 0, 0 };
    if (p.splits > 1) {
        const PartEpi e = { (int *)(base + p.part), d.m, d.n };
        const hipError_t err = k8_product<true>(g, p.tile, e, st);
        if (err != hipSuccess) return err;
        const unsigned grid = (unsigned)((d.m * ((d.n + 255) / 256) + 3) / 4);
        K8_TYPE(d.y_type, T, k8_join<T><<<dim3(grid), 256, 0, st>>>(e.part, p.splits, o));
        return hipGetLastError();
    }
    K8_TYPE(d.y_type, T, return k8_product<true>(g, p.tile, LinearEpi<T>{ o }, st));
}
