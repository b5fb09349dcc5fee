// k8_grad.hip -- the gradient of the 8-bit dense layers (include/dnascent_hip.h has the formulas).
//
// Both products have a whole-number operand (codes, exact in fp16 and in bf16) and one that carries the scales: dz sw[n] for dx, dz s[m] for dw.  That one is
// held in fp16 under a power of two of its own -- per row for dx, per output channel for dw: whatever is the same for a whole sum.  16-bit results take one
// piece, 11 bits (half a step: 2^-12 of the value; their own rounding is 2^-9 or 2^-12), fp32 results two, 22 bits: the second one is what the first left, times
// 2^12, against codes or sums times 2^-12.
// That holds for values of at least 2^-14 under their power: 2^-28 of a row's largest for dx (2^-18 where k8_dx_narrow takes an upper bound for it), 2^-24 of a
// channel's largest so far for dw.  A smaller one may be all that a result has -- the code under the large one can be zero, and half the codes behind a ReLU are --
// so whoever meets one marks its row (k8_pieces), its sixteen rows (k8_dx_narrow) or its tile (k8_dw, which leaves it out), and k8_again makes those from bf16
// pieces, whose exponents reach as far as fp32's: two for 16-bit results (2^-17), three for fp32 ones (2^-25), for values down to 2^-100.
// Sums are fp32; their order depends on the sizes and on what is marked, both the same every time.
#include "k8_dense.h"
#include "k8_dev.h"
#include <type_traits>

namespace {

typedef _Float16 k8_f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ k8_f32x4 k8_mfma16(i32x4 a, i32x4 b, k8_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(k8_f16x8, a), __builtin_bit_cast(k8_f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ int k8_pack(float a, float b) { return __builtin_bit_cast(int, k8_f16x2{ (_Float16)a, (_Float16)b }); }
__device__ __forceinline__ void k8_opaque(unsigned &v) { asm volatile("" : "+v"(v)); }
typedef __bf16 k8_bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ k8_f32x4 k8_mfma16b(i32x4 a, i32x4 b, k8_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(k8_bf16x8, a), __builtin_bit_cast(k8_bf16x8, b), c, 0, 0, 0);
}
constexpr float K8_LOW = 0x1p12f;                         // what the second fp16 piece is multiplied with
// the smallest of the magnitudes above zero, twice its bits less one: zero counts as the largest number there is
__device__ __forceinline__ unsigned k8_least(unsigned least, float v) { return min(least, (__float_as_uint(v) << 1) - 1u); }
constexpr unsigned K8_SMALL = (0x38800000u << 1) - 1u;     // 2^-14: below it fp16 has fewer bits
// two numbers in bf16 pieces; behind infinity and NaN there is nothing to add
__device__ __forceinline__ unsigned k8_bf16_pair(float v0, float v1) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    unsigned w = __builtin_bit_cast(unsigned, b2{ (__bf16)v0, (__bf16)v1 });
    asm volatile("" : "+v"(w));
    return w;
}
__device__ __forceinline__ int k8_bf16_take(float &v0, float &v1) {            // the first piece; what is left stays
    const unsigned w = k8_bf16_pair(v0, v1);
    v0 -= __uint_as_float(w << 16); v1 -= __uint_as_float(w & 0xffff0000u);
    v0 = v0 == v0 ? v0 : 0.0f; v1 = v1 == v1 ? v1 : 0.0f;
    return (int)w;
}
// eight codes in fp16 -> in bf16: the upper halves of their fp32 forms
__device__ __forceinline__ i32x4 k8_bf16_codes(i32x4 h) {
    i32x4 o;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const int w = h[p];
        const k8_f16x2 two = __builtin_bit_cast(k8_f16x2, w);
        o[p] = (int)__builtin_amdgcn_perm(__float_as_uint((float)two[1]), __float_as_uint((float)two[0]), 0x07060302u);
    }
    return o;
}
// two numbers as two fp16 pieces each, the second times 2^12.  `hi` is hidden from the compiler: left to itself it forms the fp16 value that is subtracted with an instruction that rounds
// the product behind v once, and stores the one that rounds twice.  Behind infinity and NaN there is nothing to add
struct K8Split { int hi, lo; };
__device__ __forceinline__ K8Split k8_split(float v0, float v1) {
    int hi = k8_pack(v0, v1);
    asm volatile("" : "+v"(hi));
    const k8_f16x2 h = __builtin_bit_cast(k8_f16x2, hi);
    const float l0 = (v0 - (float)h[0]) * K8_LOW, l1 = (v1 - (float)h[1]) * K8_LOW;
    return { hi, k8_pack(l0 == l0 ? l0 : 0.0f, l1 == l1 ? l1 : 0.0f) };
}
// eight rows of four codes -> four columns of eight fp16: bytes j of two rows side by side, 0x6400 | (code ^ 0x80) is 1152 + code
__device__ __forceinline__ void k8_columns(const unsigned (&d)[8], i32x4 (&out)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const unsigned t = __builtin_amdgcn_perm(d[2 * p + 1], d[2 * p], 0x0c000c00u | (unsigned)j | (unsigned)(4 + j) << 16) ^ 0x64806480u;
            out[j][p] = __builtin_bit_cast(int, __builtin_bit_cast(k8_f16x2, t) - k8_f16x2{ (_Float16)1152.0f, (_Float16)1152.0f });
        }
}
// rows first .. first + 7 of `n` rows, four codes each from channel kk of k on, without a branch around a load: rows behind the last one repeat it (what they are multiplied
// with is zero), four channels that end behind the matrix are read in front of its end and moved down
__device__ __forceinline__ void k8_eight_rows(const int8_t *__restrict__ from, int64_t ld, int64_t n, int64_t k, int64_t first, int64_t kk, unsigned (&rows)[8]) {
    if (k >= 4) {
        const int64_t at = min(kk, k - 4);
        const int skip = 8 * (int)min(kk - at, (int64_t)3);
#pragma unroll
        for (int e = 0; e < 8; e++) __builtin_memcpy(&rows[e], from + min(first + e, n - 1) * ld + at, 4);
#pragma unroll
        for (int e = 0; e < 8; e++) rows[e] >>= skip;
    } else
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int8_t *p = from + min(first + e, n - 1) * ld;
            rows[e] = 0u;
#pragma unroll
            for (int j = 0; j < 4; j++) rows[e] |= (unsigned)(uint8_t)p[min(kk + j, k - 1)] << (8 * j);
        }
}
// the power of two that puts `top` (bits of a magnitude, finite) into [2^14, 2^15), and its inverse; both are normal numbers
struct K8Pow { float up, down; };
__device__ __forceinline__ K8Pow k8_pow(unsigned top) {
    const int e = min(max(268 - (int)(top >> 23), 1), 253);
    return { __uint_as_float((unsigned)e << 23), __uint_as_float((unsigned)(254 - e) << 23) };
}

// ---- dx, narrow layers (N <= 256) ------------------------------------------------------------------------------------------------------------------------------
// The same shape as the forward pass over narrow rows (k8_narrow): a wavefront takes 16 rows of dy, holds them in registers in the matrix operand's order, finds
// each row's power of two, and multiplies with the weight, whose transposed fragments lie in LDS as fp16 (256 k x N).  Nothing but dy, the mask and dx moves.
// NP: pieces.  512 threads, so that a lane has 256 registers: enough up to N = 128, and for N = 256 all but 9 (bf16), 15 (fp16) or 58 (fp32), which go to memory; 768 threads
// hide more but keep less (100000 x 256 x 256 with dw, bf16, us: 80 : 91; 1 Mi rows, 499 : 517).
// 1 Mi x 256 x 256 bf16 with ReLU: 258 us; its 1.1 GB take 213 at a copy's rate, its products 104, and the vector instructions that mask, scale and convert about as long.
template <class T, int NS, int NP>
__global__ __launch_bounds__(512) void k8_dx_narrow(dn_i8_grad_desc d, uint8_t *__restrict__ again) {
    constexpr int WG = 512;
    __shared__ __align__(16) char lw[256 * NS * 64];       // fragment (k block of 64, tile t, step) x 64 lanes x 16 bytes: column k = 64 blk + 4 c + t, n = 32 step + 8 g ..
    __shared__ __align__(16) float lsw[NS * 32];
    __shared__ __align__(16) unsigned keep[sizeof(T) == 2 ? 256 : 1][4];      // a mask byte as eight 16-bit masks
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int n = (int)d.n;
    const int64_t k0 = (int64_t)blockIdx.y * 256;
    const int cols = (int)min((int64_t)256, d.k - k0), blocks = (cols + 63) / 64;
#pragma unroll 2
    for (int f = threadIdx.x; f < blocks * NS * 64; f += WG) {
        const int fc = f & 15, fg = (f >> 4) & 3, step = (f >> 6) % NS, blk = (f >> 6) / NS, kk = blk * 64 + 4 * fc;
        unsigned rows[8];
        k8_eight_rows(d.w, d.ldw, d.n, d.k, step * 32 + 8 * fg, k0 + kk, rows);
        i32x4 out[4];
        k8_columns(rows, out);
#pragma unroll
        for (int t = 0; t < 4; t++) *(i32x4 *)(lw + (((blk * 4 + t) * NS + step) * 64 + fg * 16 + fc) * 16) = out[t];
    }
    for (int i = threadIdx.x; i < NS * 32; i += WG) lsw[i] = i < n ? d.sw[i] : 0.0f;
    if (sizeof(T) == 2 && threadIdx.x < 256)
#pragma unroll
        for (int p = 0; p < 4; p++) keep[threadIdx.x][p] = (threadIdx.x >> 2 * p & 1 ? 0xffffu : 0u) | (threadIdx.x >> 2 * p & 2 ? 0xffff0000u : 0u);
    __syncthreads();
    // A row's power of two comes from max |dz| max |sw| -- an upper bound of its dz sw that needs no products -- unless the channels' scales are more than 2^10 apart:
    // then, and where something is not finite, from the finite dz sw themselves
    float swmost = 0.0f, swleast = 0x1.fffffep127f;
    for (int i = lane; i < n; i += 64) { const float v = fabsf(lsw[i]); swmost = fmaxf(swmost, v); if (v > 0.0f) swleast = fminf(swleast, v); }
    for (int o = 32; o; o >>= 1) { swmost = fmaxf(swmost, __shfl_xor(swmost, o)); swleast = fminf(swleast, __shfl_xor(swleast, o)); }
    const bool apart = !(swmost <= swleast * 1024.0f);
    // a lane's places behind a row's end hold no number: `real` has a bit for each that does (byte s of the pair: step s)
    unsigned real[2] = { 0u, 0u };
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const int have = min(max(n - (s * 32 + 8 * g), 0), 8);
        real[s / 4] |= ((1u << have) - 1u) << (8 * (s % 4));
    }
    K8Raw<T, 8> raw[NS];
    unsigned bit[NS];
    const bool masked = d.mask != nullptr;
    // WHOLE: seven more rows lie behind the tile, so that eight numbers can be read at once wherever a row ends (and a lane that has none there reads its row's first)
    auto fetch = [&](int64_t tile, auto kind) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(kind)::value;
        const int64_t first = tile * 16;
        const unsigned r = WHOLE ? (unsigned)c : (unsigned)min((int64_t)c, d.m - 1 - first);
        const k8_global p = k8_base((const char *)d.dy + first * d.ldy * (int64_t)sizeof(T));
        const unsigned row = r * (unsigned)d.ldy * (unsigned)sizeof(T);
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const int at = s * 32 + 8 * g;
            if (WHOLE) raw[s].load(p + (row + (unsigned)((at < n ? at : 0) * (int)sizeof(T))));
            else raw[s].load(p + (row + (unsigned)(at * (int)sizeof(T))), n - at);
        }
        if (masked) {
            const k8_global pm = k8_base(d.mask + first * d.ldmask);
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const int at = (s * 32 + 8 * g) >> 3;
                bit[s] = *(const __attribute__((address_space(1))) unsigned char *)(pm + (r * (unsigned)d.ldmask + (unsigned)(at * 8 < n ? at : 0)));
            }
        }
    };
    auto work = [&](int64_t tile, auto &&next) __attribute__((always_inline)) {
        i32x4 a[NP][NS];
        // masked numbers and places behind the row's end become zeros, in place
        if (masked || n != NS * 32)
#pragma unroll
            for (int s = 0; s < NS; s++) {
                unsigned kept = real[s / 4] >> (8 * (s % 4)) & 255u;
                if (masked) kept &= bit[s];
                if constexpr (sizeof(T) == 2) {
                    const i32x4 m = *(const i32x4 *)keep[kept];
#pragma unroll
                    for (int p = 0; p < 4; p++) raw[s].w[p] &= (unsigned)m[p];
                } else
#pragma unroll
                    for (int e = 0; e < 8; e++) raw[s].w[e] &= (unsigned)((int)(kept << (31 - e)) >> 31);
            }
        auto value = [&](int s, int e, const K8Vec<float, 8> &sw) __attribute__((always_inline)) { return raw[s].get(e) * sw.v[e]; };
        unsigned here = 8 * g;                             // hidden: the 64 factors are read again for every tile instead of being kept
        k8_opaque(here);
        float most = raw[0].most();
#pragma unroll
        for (int s = 1; s < NS; s++) most = fmaxf(most, raw[s].most());             // (of 16-bit numbers: NaN counts as infinity)
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        if (apart || __any(!(most <= 0x1.fffffep127f))) {
            most = 0.0f;
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const K8Vec<float, 8> sw = *(const K8Vec<float, 8> *)(lsw + s * 32 + here);
                raw[s].opaque();
#pragma unroll
                for (int e = 0; e < 8; e++) { const float v = fabsf(value(s, e, sw)); most = fmaxf(most, v <= 0x1.fffffep127f ? v : 0.0f); }
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
        } else most = fminf(most * swmost, 0x1.fffffep127f);
        const K8Pow pw = k8_pow(__float_as_uint(most));
        unsigned least = ~0u;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < NS; s++) {
            raw[s].opaque(); k8_opaque(here);
            const K8Vec<float, 8> sw = *(const K8Vec<float, 8> *)(lsw + s * 32 + here);
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const float v0 = value(s, 2 * p, sw) * pw.up, v1 = value(s, 2 * p + 1, sw) * pw.up;
                least = k8_least(k8_least(least, v0), v1);
                if (NP == 2) {
                    const K8Split w = k8_split(v0, v1);
                    a[0][s][p] = w.hi; a[NP - 1][s][p] = w.lo;
                } else a[0][s][p] = k8_pack(v0, v1);
            }
            // made here and now: sunk behind the next tile's loads, they would keep this tile's numbers alive beside those
#pragma unroll
            for (int p = 0; p < NP; p++) asm volatile("" : "+v"(a[p][s]));
        }
        if (blockIdx.y == 0) { const bool under = __any(least < K8_SMALL); if (lane == 0) again[tile] = under; }
        __builtin_amdgcn_sched_barrier(0);
        next();
        __builtin_amdgcn_sched_barrier(0);
        float rs[4];
#pragma unroll
        for (int q = 0; q < 4; q++) rs[q] = __shfl(pw.down, 4 * g + q);
        for (int blk = 0; blk < blocks; blk++) {
            k8_f32x4 acc[4];
            const char *lb = lw + (blk * 4 * NS * 64 + lane) * 16;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                acc[t] = k8_f32x4{ 0, 0, 0, 0 };
                k8_f32x4 low = { 0, 0, 0, 0 };
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const i32x4 b = *(const i32x4 *)(lb + (t * NS + s) * 1024);
                    acc[t] = k8_mfma16(a[0][s], b, acc[t]);
                    if (NP == 2) low = k8_mfma16(a[NP - 1][s], b, low);
                }
                if (NP == 2)
#pragma unroll
                    for (int q = 0; q < 4; q++) acc[t][q] = __builtin_fmaf(low[q], 1.0f / K8_LOW, acc[t][q]);
                __builtin_amdgcn_sched_barrier(0);         // a tile's operands at a time: more of them in flight spill
            }
            const int64_t kk = k0 + blk * 64 + 4 * c;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int64_t mm = tile * 16 + 4 * g + q;
                if (mm >= d.m || kk >= d.k) continue;
                T *p = (T *)d.dx + mm * d.ldx + kk;
                K8Vec<T, 4> o;
#pragma unroll
                for (int t = 0; t < 4; t++) o.v[t] = (T)(acc[t][q] * rs[q]);
                if (kk + 4 <= d.k) k8_stream<T, 4>(p, o);
                else
#pragma unroll
                    for (int t = 0; t < 4; t++) if (kk + t < d.k) p[t] = o.v[t];
            }
        }
    };
    const int64_t tiles = (d.m + 15) / 16, stride = (int64_t)gridDim.x * (WG / 64), whole = d.ldy ? max(d.m - 7, (int64_t)0) / 16 : 0;
    int64_t tile = (int64_t)blockIdx.x * (WG / 64) + wave;
    if (tile < whole) fetch(tile, std::true_type());
    for (; tile < whole; tile += stride) work(tile, [&]() __attribute__((always_inline)) { if (tile + stride < whole) fetch(tile + stride, std::true_type()); });
    for (; tile < tiles; tile += stride) {
        fetch(tile, std::false_type());
        work(tile, []() {});
    }
}

// ---- dx, wide layers: the pieces of dz sw as rows of fp16, the transposed weight as rows of fp16, then k8_gemm -----------------------------------------------------
// LPR lanes hold a row, V pieces of eight numbers each; with V = 0 they walk it twice (the second time from cache).  np: pitch in fp16, a multiple of 8; zeros behind n.
// Two pieces: the second one's plane comes first (k8_gemm multiplies its sums with 2^-12 where the first one's begins).
// HBM: 8192 x 4096 bf16, 23 us, 5.8 TB/s.  The weight beside it (k8_turn): 4096 x 4096, 15 us; the product: 250 us, 1.10 PFLOP/s.
template <class T, int LPR, int V, int NP>
__global__ __launch_bounds__(256) void k8_pieces(dn_i8_grad_desc d, _Float16 *__restrict__ out, int np, int64_t plane, float *__restrict__ down, uint8_t *__restrict__ again) {
    const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int lid = threadIdx.x % LPR, n = (int)d.n;
    const int64_t rr = min(row, d.m - 1);
    const T *p = (const T *)d.dy + rr * d.ldy;
    const uint8_t *mk = d.mask ? d.mask + rr * d.ldmask : nullptr;
    constexpr int HELD = V ? V : 1;
    K8Raw<T, 8> x[HELD]; K8Raw<float, 8> sw[HELD]; unsigned bits[HELD];
    float v[HELD][8];
    auto load = [&](int i, int at) __attribute__((always_inline)) {            // zeros behind the row's end
        if (at + 8 <= n) { x[i].load(p + at); sw[i].load(d.sw + at); }
        else { x[i].load(p + at, n - at); sw[i].load(d.sw + at, n - at); }
        bits[i] = mk ? mk[min(at, n - 1) >> 3] : 255u;
    };
    auto make = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] = __uint_as_float(__float_as_uint(x[i].get(e)) & (unsigned)((int)(bits[i] << (31 - e)) >> 31)) * sw[i].get(e);
    };
    unsigned top = 0;
    auto most = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++) { const unsigned b = k8_mag(v[i][e]); top = max(top, b < 0x7f800000u ? b : 0u); }
    };
    if (V) {
#pragma unroll
        for (int i = 0; i < V; i++) load(i, (i * LPR + lid) * 8);
#pragma unroll
        for (int i = 0; i < V; i++) { make(i); most(i); }
    } else
        for (int at = lid * 8; at < n; at += LPR * 8) { load(0, at); make(0); most(0); }
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    if (LPR == 256) {
        __shared__ unsigned part[4];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    if (row >= d.m) return;
    const K8Pow pw = k8_pow(top);
    if (lid == 0) down[row] = pw.down;
    unsigned least = ~0u;
    auto store = [&](int i, int at) __attribute__((always_inline)) {
        i32x4 hi, lo;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float v0 = v[i][2 * q] * pw.up, v1 = v[i][2 * q + 1] * pw.up;
            least = k8_least(k8_least(least, v0), v1);
            if (NP == 2) { const K8Split w = k8_split(v0, v1); hi[q] = w.hi; lo[q] = w.lo; }
            else hi[q] = k8_pack(v0, v1);
        }
        *(i32x4 *)(out + (NP - 1) * plane + row * np + at) = hi;
        if (NP == 2) *(i32x4 *)(out + row * np + at) = lo;
    };
    if (V) {
#pragma unroll
        for (int i = 0; i < V; i++) if ((i * LPR + lid) * 8 < np) store(i, (i * LPR + lid) * 8);
    } else
        for (int at = lid * 8; at < np; at += LPR * 8) { load(0, at); make(0); store(0, at); }
    const bool under = LPR == 256 ? __syncthreads_or(least < K8_SMALL) : __any(least < K8_SMALL);
    if (lid == 0) again[row] = under;
}
// w [n][k] codes -> [k][np] fp16, zeros behind n.  A thread takes 8 n x 4 k; the 8 lanes beside it the next 64 n
__global__ __launch_bounds__(256) void k8_turn(dn_i8_grad_desc d, _Float16 *__restrict__ out, int np) {
    const int k = (int)d.k;
    const int64_t nb = (np + 63) / 64, kb = (k + 127) / 128;
    const int64_t bn = blockIdx.x % nb, bk = blockIdx.x / nb;
    if (bk >= kb) return;
    const int nn = (int)bn * 64 + (threadIdx.x & 7) * 8, kk = (int)bk * 128 + (threadIdx.x >> 3) * 4;
    if (nn >= np || kk >= k) return;
    unsigned rows[8];
    k8_eight_rows(d.w, d.ldw, d.n, d.k, nn, kk, rows);
    i32x4 o[4];
    k8_columns(rows, o);
#pragma unroll
    for (int j = 0; j < 4; j++) if (kk + j < k) *(i32x4 *)(out + (int64_t)(kk + j) * np + nn) = o[j];
}
template <class T>
struct DxEpi {
    typedef float value;
    const float *down; T *dx; int64_t k, ldx;
    template <int TN> struct Columns {};
    template <int TN> __device__ __forceinline__ Columns<TN> columns(int64_t) const { return {}; }
    template <int TN> struct Row { float down; };
    template <int TN> __device__ __forceinline__ Row<TN> row(int64_t mm, int64_t) const { return { down[mm] }; }
    template <int TN> __device__ __forceinline__ void store(const Columns<TN> &, const Row<TN> &r, int64_t mm, int64_t kk, int, const float (&acc)[TN], bool live) const {
        if (!live) return;
        T *p = dx + mm * ldx + kk;
        K8Vec<T, TN> o;
#pragma unroll
        for (int j = 0; j < TN; j++) o.v[j] = (T)(acc[j] * r.down);
        if (kk + TN <= k) k8_stream<T, TN>(p, o);
        else
#pragma unroll
            for (int j = 0; j < TN; j++) if (kk + j < k) p[j] = o.v[j];
    }
};
// a run's sums: part [splits][m][k]
struct DxPart {
    typedef float value;
    float *part; int64_t m, k;
    template <int TN> struct Columns {};
    template <int TN> __device__ __forceinline__ Columns<TN> columns(int64_t) const { return {}; }
    template <int TN> struct Row {};
    template <int TN> __device__ __forceinline__ Row<TN> row(int64_t, int64_t) const { return {}; }
    template <int TN> __device__ __forceinline__ void store(const Columns<TN> &, const Row<TN> &, int64_t mm, int64_t kk, int z, const float (&acc)[TN], bool live) const {
        if (!live) return;
        float *p = part + ((int64_t)z * m + mm) * k + kk;
#pragma unroll
        for (int j = 0; j < TN; j++) if (kk + j < k) p[j] = acc[j];
    }
};
template <class T>
__global__ __launch_bounds__(256) void k8_dx_join(const float *__restrict__ part, int splits, const float *__restrict__ down, T *__restrict__ dx, int64_t m, int64_t k, int64_t ldx) {
    const int64_t kb = (k + 255) / 256, w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= m * kb) return;
    const int64_t mm = w / kb, kk = (w % kb) * 256 + (threadIdx.x & 63) * 4, left = k - kk;
    if (left <= 0) return;
    float v[4] = { 0, 0, 0, 0 };
    const float *p = part + mm * k + kk;
    if (left >= 4)
#pragma unroll 8
        for (int z = 0; z < splits; z++) {
            const K8Vec<float, 4> t = k8_load<float, 4>(p + (int64_t)z * m * k);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += t.v[j];
        }
    else
        for (int z = 0; z < splits; z++)
#pragma unroll
            for (int j = 0; j < 3; j++) if (j < left) v[j] += p[(int64_t)z * m * k + j];
    const float s = down ? down[mm] : 1.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] *= s;
    T *o = dx + mm * ldx + kk;
    K8Vec<T, 4> y;
#pragma unroll
    for (int j = 0; j < 4; j++) y.v[j] = (T)v[j];
    if (left >= 4) k8_store<T, 4>(o, y);
    else
#pragma unroll
        for (int j = 0; j < 3; j++) if (j < left) o[j] = y.v[j];
}

// ---- dx, few rows (M <= 16): the weight is streamed once, turned in registers -------------------------------------------------------------------------------------
// A workgroup takes 64 input channels; its eight wavefronts deal the output channels among themselves, 64 at a time, and join their sums in LDS.  A lane reads
// eight rows of four codes and makes the operands of the four column tiles of them.  Each 64 numbers of a row have a power of two of their own, so nothing has to
// be known of a row before the weight's first bytes are asked for; its factors are bf16 pieces (there is time for all of them while the weight is on its way).
// Where that makes few workgroups for many output channels, the output channels are cut into runs of `run` as well, and k8_dx_join adds the runs' results.
// Bound by latency: 6 x 1991 x 3807 fp16 11 us, 7 x 16384 x 1024 bf16 9 + 5 us (one run: 54), 12 x 4096 x 4096 9 + 3.
template <class T> struct K8Few {                          // 64 numbers of sixteen rows, and what comes of them
    static constexpr int PIECES = sizeof(T) == 4 ? 3 : 2;
    K8Raw<T, 8> x[2]; K8Raw<float, 8> sw[2]; unsigned bits[2];
    i32x4 a[2][PIECES]; float down;
    __device__ __forceinline__ void pieces(bool masked) {
        float v[2][8], most = 0.0f;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float z = x[s].get(e);
                if (masked) z = __uint_as_float(__float_as_uint(z) & (unsigned)((int)(bits[s] << (31 - e)) >> 31));
                v[s][e] = z * sw[s].get(e);
                most = fmaxf(most, fabsf(v[s][e]));
            }
        if (__any(!(most <= 0x1.fffffep127f))) {           // the largest finite one
            most = 0.0f;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int e = 0; e < 8; e++) { const float f = fabsf(v[s][e]); most = fmaxf(most, f <= 0x1.fffffep127f ? f : 0.0f); }
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const K8Pow pw = k8_pow(__float_as_uint(most));
        down = pw.down;
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int p = 0; p < 4; p++) {
                float v0 = v[s][2 * p] * pw.up, v1 = v[s][2 * p + 1] * pw.up;
#pragma unroll
                for (int i = 0; i < PIECES; i++) a[s][i][p] = k8_bf16_take(v0, v1);
            }
    }
    // b: codes in bf16
    __device__ __forceinline__ void add(const i32x4 (&b)[2][4], k8_f32x4 (&sum)[4]) const {
        const int g = (threadIdx.x & 63) >> 4;
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __shfl(down, 4 * g + i);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            k8_f32x4 acc = { 0, 0, 0, 0 };
#pragma unroll
            for (int i = PIECES - 1; i >= 0; i--)          // the small ones first
#pragma unroll
                for (int s = 0; s < 2; s++) acc = k8_mfma16b(a[s][i], b[s][t], acc);
#pragma unroll
            for (int i = 0; i < 4; i++) sum[t][i] = __builtin_fmaf(acc[i], f[i], sum[t][i]);
        }
    }
};
// eight wavefronts' sums joined: put(row, column of 64, value)
template <class Put> __device__ __forceinline__ void k8_few_join(float (&sums)[8][4][256], const k8_f32x4 (&sum)[4], int m, int cols, Put &&put) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 4; t++)                            // D: column lane & 15, row 4 g + i
#pragma unroll
        for (int i = 0; i < 4; i++) sums[wave][t][(4 * g + i) * 16 + c] = sum[t][i];
    __syncthreads();
    const int kk = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < m; r += 8) {
        float v = 0.0f;
#pragma unroll
        for (int z = 0; z < 8; z++) v += sums[z][kk & 3][r * 16 + (kk >> 2)];
        if (kk < cols) put(r, kk, v);
    }
}
template <class T>
__global__ __launch_bounds__(512) void k8_dx_few(dn_i8_grad_desc d, int run, float *part) {
    __shared__ __align__(16) float sums[8][4][256];
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4, n = (int)d.n, m = (int)d.m;
    const int64_t k0 = (int64_t)blockIdx.x * 64;
    const int64_t row = min(c, m - 1);                     // operand rows behind the last one repeat it
    K8Few<T> f;
    unsigned rows[2][8];
    const T *px = (const T *)d.dy + row * d.ldy + 8 * g;
    const uint8_t *pm = d.mask ? d.mask + row * d.ldmask : nullptr;
    // four columns that end behind the matrix are read in front of its end and moved down
    const int64_t at_k = min(k0 + 4 * c, d.k - 4);
    const int down8 = 8 * (int)min(k0 + 4 * c - at_k, (int64_t)3);
    const unsigned ldw = (unsigned)d.ldw, pw0 = (unsigned)(8 * g) * ldw + (unsigned)at_k;
    typedef const __attribute__((address_space(1))) k8_u32 *gu32;
    auto fetch = [&](int step, auto kind) __attribute__((always_inline)) {     // WHOLE: the row does not end here
        constexpr bool WHOLE = decltype(kind)::value;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int at0 = step * 64 + s * 32, at = at0 + 8 * g;
            if (WHOLE) { f.x[s].load(px + at0); f.sw[s].load(d.sw + at); }
            else { f.x[s].load(px + at0, n - at); f.sw[s].load(d.sw + at, n - at); }
            if (pm) f.bits[s] = pm[min(at, n - 1) >> 3];
            const k8_global w = k8_base(d.w + at0 * d.ldw);
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (WHOLE) rows[s][e] = *(gu32)(w + e * (int64_t)ldw + pw0);
                else rows[s][e] = *(gu32)(k8_base(d.w) + (int64_t)min(at + e, n - 1) * ldw + at_k);            // zeros times the last row behind the end
        }
    };
    k8_f32x4 sum[4];
#pragma unroll
    for (int t = 0; t < 4; t++) sum[t] = k8_f32x4{ 0, 0, 0, 0 };
    const int steps = (min(n, ((int)blockIdx.y + 1) * run) + 63) / 64;         // (a run is whole steps)
    auto next = [&](int step) __attribute__((always_inline)) {
        if (step < steps && step * 64 + 64 <= n) fetch(step, std::true_type());
        else if (step < steps) fetch(step, std::false_type());
    };
    const int first = (int)blockIdx.y * (run / 64) + wave;
    next(first);
    for (int step = first; step < steps; step += 8) {
        i32x4 b[2][4];
        f.pieces(pm);
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int e = 0; e < 8; e++) rows[s][e] >>= down8;
            k8_columns(rows[s], b[s]);
#pragma unroll
            for (int t = 0; t < 4; t++) b[s][t] = k8_bf16_codes(b[s][t]);
        }
        next(step + 8);
        f.add(b, sum);
    }
    k8_few_join(sums, sum, m, (int)min((int64_t)64, d.k - k0), [&](int r, int kk, float v) __attribute__((always_inline)) {
        if (part) part[((int64_t)blockIdx.y * m + r) * d.k + k0 + kk] = v;
        else ((T *)d.dx)[r * d.ldx + k0 + kk] = (T)v;
    });
}

// ---- dw and db --------------------------------------------------------------------------------------------------------------------------------------------------
// The reduction runs over rows, along which neither operand is contiguous.  A workgroup takes S x S results (output channels x input channels) and a run of rows,
// RT at a time: a thread reads eight rows of four adjacent channels, makes the fp16 values and writes them to LDS turned -- eight rows of one channel are the
// 16 bytes a matrix instruction takes.  The rows of the next tile are in flight while this one multiplies.
//
// Every output channel has a power of two, agreed on by the whole workgroup: it comes from the largest numbers of the first tile, with five bits of room.  Whoever sees
// a number that does not fit raises a flag; behind the barrier the workgroup then finds that tile's largest numbers, lowers the powers of the channels that need it,
// scales their sums so far -- exactly -- and makes the tile again, which hardly ever happens.
//
// LDS row of a channel: RT rows x 2 bytes (x NP pieces), in pieces of 16 bytes.  Threads that write and lanes that read stand four channels apart: those lie side by side, and
// sixteen of them reach sixteen different places of the 64 banks.  Wavefronts share the S x S results in blocks of 64 x KB; where there are fewer blocks than wavefronts, sets of wavefronts take turns
// with the steps of 32 rows and join their sums at the end.
template <int S, int NP> struct DwShape {
    static constexpr int RT = 16384 / S / NP;              // rows of a tile: S = 256: 64, 128: 128, 64: 256 (half with two pieces)
    static constexpr int KB = S == 256 ? 128 : 64, BLOCKS = (S / 64) * (S / KB), SETS = 8 / BLOCKS, STEPS = RT / 32;
    static constexpr int UROW = RT * 2 * NP, QROW = UROW;   // bytes of a channel's row; two pieces: the codes as they are and times 2^-12
    static constexpr int LDS = S * (UROW + QROW);           // one stage
};
template <int ROW> __device__ __forceinline__ int k8_place(int block, int i, int c, int piece) {      // channel 64 block + 4 c + i; ROW: bytes of a channel's row
    return (block * 64 + i * 16 + c) * ROW + ((piece ^ (ROW >= 256 ? c : ROW == 128 ? c >> 1 : c >> 2)) << 4);
}
// part [splits][n][k], part_b [splits][n]; run: rows of a split, a multiple of RT; again [blocks of 64 output channels][row_tiles]: which tiles were left out.  A single
// split puts results that lack some into part as well
struct DwOut { float *part, *part_b; int splits, tiles_n, tiles_k; int64_t run; uint8_t *again; int64_t row_tiles; };

template <class W> __device__ __forceinline__ void k8_put4(W *p, const float (&v)[4], int64_t left) {
    K8Vec<W, 4> o;
#pragma unroll
    for (int j = 0; j < 4; j++) o.v[j] = (W)v[j];
    if (left >= 4) k8_store<W, 4>(p, o);
    else
#pragma unroll
        for (int j = 0; j < 4; j++) if (j < left) p[j] = o.v[j];
}
__device__ __forceinline__ void k8_put4(void *p, int type, int64_t at, const float (&v)[4], int64_t left) {
    if (type == DN_T_F32) k8_put4((float *)p + at, v, left);
    else if (type == DN_T_F16) k8_put4((_Float16 *)p + at, v, left);
    else k8_put4((k8_bf16 *)p + at, v, left);
}

__device__ __forceinline__ void k8_put1(void *p, int type, int64_t at, float v) {
    if (type == DN_T_F32) ((float *)p)[at] = v;
    else if (type == DN_T_F16) ((_Float16 *)p)[at] = (_Float16)v;
    else ((k8_bf16 *)p)[at] = (k8_bf16)v;
}

template <class T, int S, int NP>
__global__ __launch_bounds__(512) void k8_dw(dn_i8_grad_desc d, DwOut o) {
    typedef DwShape<S, NP> D;
    __shared__ __align__(1024) char lds[2][D::LDS];
    __shared__ __align__(16) float power[S], lower[S];
    __shared__ unsigned peak[S];
    // of a tile (they take turns: one is cleared while the one before it is read): bit 0, a value that does not fit; bit 1 + b, one in block b of 64 output channels that
    // is too small for fp16
    __shared__ unsigned flags[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = k8_uniform(tid >> 6), c = lane & 15, g = lane >> 4;
    const int tiles = o.tiles_n * o.tiles_k, z = blockIdx.x / tiles, t = blockIdx.x % tiles, tn = t % o.tiles_n, tk = t / o.tiles_n;
    const int64_t n0 = (int64_t)tn * S, k0 = (int64_t)tk * S, r0 = (int64_t)z * o.run, r1 = min(r0 + o.run, d.m);
    const int ncols = (int)min((int64_t)S, d.n - n0), kcols = (int)min((int64_t)S, d.k - k0);
    const bool with_q = d.dw != nullptr, with_b = d.db != nullptr && tk == 0;
    for (int i = tid; i < S; i += 512) power[i] = 0x1p126f;
    if (tid < 3) flags[tid] = 0u;
    __syncthreads();
    // a task: eight rows x four channels.  S / 4 tasks across, RT / 8 down; with RT S = 16384 / NP that is 512 / NP for each of dy and q: one per thread, or with two
    // pieces dy's for the first four wavefronts and q's for the others
    constexpr int ACROSS = S / 4, TASKS = ACROSS * (D::RT / 8);
    static_assert(TASKS == 512 / NP, "one task per thread");
    const bool has_u = tid < TASKS, has_q = NP == 1 || tid >= TASKS;
    const int task = NP == 1 ? tid : tid & (TASKS - 1), ch = (task % ACROSS) * 4, rg = task / ACROSS;      // first channel, group of eight rows
    K8Raw<T, 4> raw[8];
    unsigned own[NP == 1 ? 8 : 1], rbit[8];
    // a row's four codes: two pieces -- dy's rows and q's are read by different wavefronts, into the same registers
    auto rq = [&](int e) __attribute__((always_inline)) -> unsigned & { if constexpr (NP == 1) return own[e]; else return raw[e].w[0]; };
    // the rows' scales.  In tiles of 256 a wavefront's lanes have the same eight rows: lane i holds the scale of row i & 7, in one register for eight
    constexpr bool ONE = S == 256;
    float rs[ONE ? 1 : 8];
    auto scale = [&](int e) __attribute__((always_inline)) {
        if constexpr (ONE) return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(rs[0]), e));
        else return rs[e];
    };
    // Two ways to fetch a tile.  WHOLE: all its rows are there and three more behind them, so that four channels can be read at once wherever a row ends (what lies
    // behind it belongs to channels that are not stored); a lane's offset leads to its group's first row, the others follow by the base.  Otherwise row by row and
    // channel by channel where a row ends; rows behind the run repeat its last one and count as zeros (no mask bit, no scale).
    const bool u_in = has_u && ch < ncols, q_in = has_q && with_q && ch < kcols;
    const int esh = (int)((n0 + ch) & 7);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        rbit[e] = ch < ncols ? 255u : 0u; rs[ONE ? 0 : e] = 0.0f; if (NP == 1) own[NP == 1 ? e : 0] = 0u;
#pragma unroll
        for (unsigned j = 0; j < sizeof(T); j++) raw[e].w[j] = 0u;
    }
    typedef const __attribute__((address_space(1))) unsigned char *gu8;
    typedef const __attribute__((address_space(1))) float *gf32;
    auto fetch = [&](int64_t base, auto kind) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(kind)::value;
        const int left = (int)min(r1 - base, (int64_t)D::RT) - 1;
        auto row = [&](int e) { return WHOLE ? (unsigned)(rg * 8) : (unsigned)min(rg * 8 + e, left); };
        auto up = [&](int e) { return WHOLE ? (int64_t)e : (int64_t)0; };
        if (u_in) {
            const k8_global pu = k8_base((const char *)d.dy + (base * d.ldy + n0) * (int64_t)sizeof(T));
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const k8_global p = pu + up(e) * d.ldy * (int64_t)sizeof(T) + (row(e) * (unsigned)d.ldy + (unsigned)ch) * (unsigned)sizeof(T);
                if (WHOLE || ncols == S) raw[e].load(p);
                else raw[e].load(p, ncols - ch);
            }
            if (d.mask) {
                const k8_global pm = k8_base(d.mask + base * d.ldmask + (n0 >> 3));
#pragma unroll
                for (int e = 0; e < 8; e++) rbit[e] = (unsigned)*(gu8)(pm + up(e) * d.ldmask + (row(e) * (unsigned)d.ldmask + (unsigned)(ch >> 3)));
            }
            if (!ONE && with_q) {
                const k8_global ps = k8_base(d.s + base);
#pragma unroll
                for (int e = 0; e < 8; e++) rs[ONE ? 0 : e] = *(gf32)(ps + up(e) * 4 + row(e) * 4u);
            }
        }
        if (ONE && with_q) rs[0] = *(gf32)(k8_base(d.s + base) + (unsigned)min(rg * 8 + (lane & 7), left) * 4u);
        if (q_in) {
            const k8_global pq = k8_base(d.q + base * d.ldq + k0);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const k8_global p = pq + up(e) * d.ldq + (row(e) * (unsigned)d.ldq + (unsigned)ch);
                if (WHOLE || kcols == S) rq(e) = *(const __attribute__((address_space(1))) k8_u32 *)p;
                else {                                     // (channels behind the last one repeat it; they are not stored)
                    rq(e) = 0u;
#pragma unroll
                    for (int j = 0; j < 4; j++) rq(e) |= (unsigned)((gu8)p)[min(j, kcols - 1 - ch)] << (8 * j);
                }
            }
        }
        if (!WHOLE) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (rg * 8 + e > left) { rbit[e] = 0u; if (!ONE) rs[ONE ? 0 : e] = 0.0f; }
                else if (!d.mask) rbit[e] = ch < ncols ? 255u : 0u;
            if (ONE && rg * 8 + (lane & 7) > left) rs[0] = 0.0f;
        }
    };
    float sum[4] = { 0, 0, 0, 0 };
    auto dz = [&](int e, int j) { return __uint_as_float(__float_as_uint(raw[e].get(j)) & (unsigned)((int)(rbit[e] << (31 - j)) >> 31)); };       // rbit: from this thread's first channel on
    // the turned fp16 values of this thread's task (and, if asked for, the sums of dz); whether one does not fit, and whether one is too small for fp16
    struct Fit { bool over, under; };
    auto make = [&](char *l, auto masked, auto sums) __attribute__((always_inline)) -> Fit {
        float most = 0.0f;
        unsigned least = ~0u;
        const k8_f32x4 pw = *(const k8_f32x4 *)(power + ch);
        if (has_u) {
            if (decltype(masked)::value)
#pragma unroll
                for (int e = 0; e < 8; e++) rbit[e] >>= esh;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                i32x4 hi, lo;
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const float z0 = decltype(masked)::value ? dz(2 * p, j) : raw[2 * p].get(j), z1 = decltype(masked)::value ? dz(2 * p + 1, j) : raw[2 * p + 1].get(j);
                    const float v0 = z0 * scale(2 * p) * pw[j], v1 = z1 * scale(2 * p + 1) * pw[j];
                    if (decltype(sums)::value) sum[j] = sum[j] + z0 + z1;
                    most = fmaxf(fmaxf(fabsf(v0), fabsf(v1)), most);
                    least = k8_least(k8_least(least, v0), v1);
                    if (NP == 2) { const K8Split w = k8_split(v0, v1); hi[p] = w.hi; lo[p] = w.lo; }
                    else hi[p] = k8_pack(v0, v1);
                }
                *(i32x4 *)(l + k8_place<D::UROW>(ch >> 6, j, ch >> 2 & 15, rg)) = hi;
                if (NP == 2) *(i32x4 *)(l + k8_place<D::UROW>(ch >> 6, j, ch >> 2 & 15, rg + D::RT / 8)) = lo;
            }
            if (decltype(masked)::value)
#pragma unroll
                for (int e = 0; e < 8; e++) rbit[e] <<= esh;
        }
        return { most > 32768.0f, least < K8_SMALL };
    };
    auto make_q = [&](char *l) __attribute__((always_inline)) {
        if (!has_q) return;
        i32x4 out[4];
        const unsigned rows[8] = { rq(0), rq(1), rq(2), rq(3), rq(4), rq(5), rq(6), rq(7) };
        k8_columns(rows, out);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            *(i32x4 *)(l + S * D::UROW + k8_place<D::QROW>(ch >> 6, j, ch >> 2 & 15, rg)) = out[j];
            if (NP == 2)                                   // (codes times 2^-12 are normal numbers in fp16)
                *(i32x4 *)(l + S * D::UROW + k8_place<D::QROW>(ch >> 6, j, ch >> 2 & 15, rg + D::RT / 8)) = __builtin_bit_cast(i32x4, __builtin_bit_cast(k8_f16x8, out[j]) * (_Float16)(1.0f / K8_LOW));
        }
    };
    const int block = wave % D::BLOCKS, set = wave / D::BLOCKS, bn = block % (S / 64), bk = block / (S / 64);
    constexpr int TK = D::KB / 16;
    k8_f32x4 acc[4][TK];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < TK; j++) acc[i][j] = k8_f32x4{ 0, 0, 0, 0 };
    // tile i of a block of 64 holds channels 4 c + i.  PART: the operands that are read at once; tiles of 256 have registers for all of them only where dy is bf16
    constexpr int PART = S < 256 || __is_same(T, k8_bf16) ? TK : sizeof(T) == 2 ? TK / 2 : TK / 4;
    auto multiply = [&](const char *l) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < (D::STEPS * NP + D::SETS - 1) / D::SETS; w++) {
            const int item = w * D::SETS + set, step = item % D::STEPS, plane = item / D::STEPS;
            if (D::STEPS * NP % D::SETS && item >= D::STEPS * NP) break;
            i32x4 a[4], b[PART];
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = *(const i32x4 *)(l + k8_place<D::UROW>(bn, i, c, plane * (D::RT / 8) + step * 4 + g));
#pragma unroll
            for (int h = 0; h < TK; h += PART) {
#pragma unroll
                for (int j = 0; j < PART; j++)
                    b[j] = *(const i32x4 *)(l + S * D::UROW + k8_place<D::QROW>(bk * (D::KB / 64) + (h + j) / 4, j % 4, c, plane * (D::RT / 8) + step * 4 + g));
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < PART; j++) acc[i][h + j] = k8_mfma16(a[i], b[j], acc[i][h + j]);
                if (PART < TK) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    int stage = 0, turn = 0;                               // turn: the tile's word of flags
    unsigned left_out = 0;                                 // blocks of 64 output channels that lack a tile
    uint8_t *mark = o.again + (int64_t)tn * (S / 64) * o.row_tiles + r0 / D::RT;           // the tile's, of the first block of 64 output channels
    // the channels' powers from the tile in hand (its mask bits already shifted down if `down`), lowered where it does not fit; power and lower are set
    auto lower_powers = [&](int down) __attribute__((always_inline)) {
        for (int i = tid; i < S; i += 512) peak[i] = 0u;
        __syncthreads();
        if (tid == 0) flags[turn] = 0u;
        if (u_in)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                unsigned top = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) { const unsigned v = k8_mag((rbit[e] >> (down + j) & 1 ? raw[e].get(j) : 0.0f) * scale(e)); top = max(top, v < 0x7f800000u ? v : 0u); }
                atomicMax(&peak[ch + j], top);
            }
        __syncthreads();
        for (int i = tid; i < S; i += 512) {
            const float was = power[i], a = __uint_as_float(peak[i]);
            float now = was;
            if (a * was > 32768.0f) now = __uint_as_float((unsigned)min(max(264 - (int)(peak[i] >> 23), 1), 253) << 23);     // a -> [2^10, 2^11)
            power[i] = now;
            lower[i] = now / was;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; e++) raw[e].opaque();       // made into numbers again by make(): kept, they would not fit the registers
    };
    // again, next: fetch this tile / the next one
    auto tile = [&](auto whole, auto &&again, auto &&next) __attribute__((always_inline)) {
        char *l = lds[stage];
        Fit fit;
        if (!decltype(whole)::value) fit = make(l, std::true_type(), std::true_type());
        else if (d.mask) fit = with_b ? make(l, std::true_type(), std::true_type()) : make(l, std::true_type(), std::false_type());
        else fit = with_b ? make(l, std::false_type(), std::true_type()) : make(l, std::false_type(), std::false_type());
        if (with_q) {
            make_q(l);
            if (fit.over || fit.under) atomicOr(&flags[turn], (fit.over ? 1u : 0u) | (fit.under ? 2u << (ch >> 6) : 0u));
            const int after = turn == 2 ? 0 : turn + 1;
            if (tid == 0) flags[after] = 0u;
            next();
            __syncthreads();
            unsigned flag = (unsigned)k8_uniform((int)flags[turn]);
            if (__builtin_expect(flag & 1u, 0)) {
                again();
                lower_powers(esh);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const float f = lower[bn * 64 + 4 * (4 * g + q) + i];
#pragma unroll
                        for (int j = 0; j < TK; j++) acc[i][j][q] *= f;
                    }
                if (make(l, std::true_type(), std::false_type()).under) atomicOr(&flags[turn], 2u << (ch >> 6));
                next();
                __syncthreads();
                flag = (unsigned)k8_uniform((int)flags[turn]);
            }
            if (tk == 0 && wave == 0) { int b = lane; asm volatile("" : "+v"(b)); if (b < S / 64) mark[b * o.row_tiles] = flag >> (1 + b) & 1u; }
            mark++;
            if (__builtin_expect(flag >> 1, 0)) {          // left out: zeros.  (Its products are made all the same: a branch around them takes 60 registers to memory)
                left_out |= flag >> 1;
                __syncthreads();
                for (int i = tid; i < S * D::UROW / 16; i += 512) if (flag >> (1 + i / (64 * D::UROW / 16)) & 1u) *(i32x4 *)(l + i * 16) = i32x4{ 0, 0, 0, 0 };
                __syncthreads();
            }
            multiply(l);
            turn = after;
        } else next();
        stage ^= 1;
    };
    // (a call without rows has one empty run: its sums are zeros)
    int64_t base = r0;
    const int64_t whole = min(r1, d.ldy && d.ldq ? d.m - 3 : (int64_t)0) - D::RT;         // the last tile that can be fetched whole starts here or before
    if (base <= whole) {
        fetch(base, std::true_type());
        if (with_q) lower_powers(esh);
    }
    for (; base <= whole; base += D::RT) tile(std::true_type(), [&]() __attribute__((always_inline)) { fetch(base, std::true_type()); },
                                                        [&]() __attribute__((always_inline)) { if (base + D::RT <= whole) fetch(base + D::RT, std::true_type()); });
    for (; base < r1; base += D::RT) {
        fetch(base, std::false_type());
        if (with_q && base == r0) lower_powers(esh);
        tile(std::false_type(), [&]() __attribute__((always_inline)) { fetch(base, std::false_type()); }, []() {});
    }
    // ---- the sums leave: sets of wavefronts joined in LDS first, half of the sets to the other half
    __syncthreads();
    const bool last = o.splits == 1;
    if (with_q) {
        float *js = (float *)lds;                          // [sets / 2][blocks][4 * TK][64] x 4 floats
        static_assert((D::SETS & (D::SETS - 1)) == 0 && D::SETS / 2 * D::BLOCKS * 4 * TK * 1024 <= 2 * D::LDS, "half of the sets' sums fit the stages");
        for (int half = D::SETS / 2; half; half /= 2) {
            if (set >= half && set < 2 * half)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < TK; j++) *(k8_f32x4 *)(js + ((((set - half) * D::BLOCKS + block) * 4 + i) * TK + j) * 256 + lane * 4) = acc[i][j];
            __syncthreads();
            if (set < half)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < TK; j++) acc[i][j] += *(const k8_f32x4 *)(js + (((set * D::BLOCKS + block) * 4 + i) * TK + j) * 256 + lane * 4);
            __syncthreads();
        }
        if (set == 0)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int cn = bn * 64 + 4 * (4 * g + q) + i;
                    if (cn >= ncols) continue;
                    const float f = 1.0f / power[cn];
#pragma unroll
                    for (int j = 0; j < TK / 4; j++) {
                        const int ck = bk * D::KB + j * 64 + 4 * c;
                        if (ck >= kcols) continue;
                        const float v[4] = { acc[i][4 * j][q] * f, acc[i][4 * j + 1][q] * f, acc[i][4 * j + 2][q] * f, acc[i][4 * j + 3][q] * f };
                        if (last && !(left_out >> bn & 1u)) k8_put4(d.dw, d.dw_type, (n0 + cn) * d.lddw + k0 + ck, v, kcols - ck);
                        else k8_put4(o.part + ((int64_t)z * d.n + n0 + cn) * d.k + k0 + ck, v, kcols - ck);
                    }
                }
        __syncthreads();
    }
    if (with_b) {
        float *js = (float *)lds;                          // [RT / 8][S]
        if (has_u)
#pragma unroll
            for (int j = 0; j < 4; j++) js[rg * S + ch + j] = sum[j];
        __syncthreads();
        for (int i = tid; i < ncols; i += 512) {
            float v = 0.0f;
            for (int r = 0; r < D::RT / 8; r++) v += js[r * S + i];
            if (!last) o.part_b[(int64_t)z * d.n + n0 + i] = v;
            else k8_put1(d.db, d.dw_type, n0 + i, v);
        }
    }
}
// ---- what fp16 has too few bits for, from bf16 pieces ---------------------------------------------------------------------------------------------------------------
// One launch behind dx's and dw's, for the rows and tiles that they marked.  Ordinary gradients mark few (normal numbers, row sizes spread by a factor of e: 3 of 2000
// tiles of 64 rows x 64 channels, next to no rows).  Bound by latency: nothing marked 2 to 5 us, 1 Mi x 256 x 256 24 us, 8192 x 4096 x 4096 35 us, both bf16.  With everything
// marked (numbers spread evenly over 2^40) the whole gradient takes 3.3 ms and 5.5 ms instead of 0.54 and 0.66, of 100000 x 256 x 256 fp32 0.46 instead of 0.15.
// dx: a workgroup takes 64 input channels and a slice of the marks, sixteen marked rows at a time (its wavefronts deal the output channels among themselves, or the
// marks if there are few channels), with k8_dx_few's arithmetic.
// dw: a workgroup takes 64 x 256 results of one run, adds up its marked tiles in steps of 64 rows, and adds that to the run's result.
struct K8Again {
    const uint8_t *dx; int rows; int64_t units; unsigned cols, slices, dx_blocks;         // a mark of dx stands for `rows` rows
    DwOut o; int rt, pieces; unsigned blocks_n, blocks_k;  // dw: tiles of rt rows; blocks of 64 output channels, of 256 input channels
};
constexpr int K8_MARKS = 512;
// which of the `n` marks from p on are set, at most K8_MARKS of them looked at: their places in order, and how many
__device__ __forceinline__ int k8_marks(const uint8_t *p, int64_t n, int *lst, int *before) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool set = tid < n && p[tid];
    if (!__syncthreads_or(set)) return 0;
    const uint64_t all = __ballot(set);
    if (lane == 0) before[wave] = __popcll(all);
    __syncthreads();
    int at = __popcll(all & ((1ull << lane) - 1)), sum = 0;
    for (int w = 0; w < 8; w++) { if (w < wave) at += before[w]; sum += before[w]; }
    if (set) lst[at] = tid;
    __syncthreads();
    return k8_uniform(sum);
}
template <class T>
__device__ __forceinline__ void k8_dx_again(const dn_i8_grad_desc &d, const K8Again &a, float (&sums)[8][4][256], int *lst, int *before) {
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4, n = (int)d.n;
    const int64_t k0 = (int64_t)(blockIdx.x % a.cols) * 64, per = (a.units + a.slices - 1) / a.slices, u0 = (blockIdx.x / a.cols) * per, u1 = min(u0 + per, a.units);
    // sixteen rows (a lane's is `row`) times the output channels of steps first, first + stride, ..
    auto product = [&](int64_t row, int first, int stride, k8_f32x4 (&sum)[4]) __attribute__((always_inline)) {
        const T *px = (const T *)d.dy + row * d.ldy;
        const uint8_t *pm = d.mask ? d.mask + row * d.ldmask : nullptr;
        K8Few<T> f;
#pragma unroll
        for (int t = 0; t < 4; t++) sum[t] = k8_f32x4{ 0, 0, 0, 0 };
        for (int step = first; step * 64 < n; step += stride) {
            i32x4 b[2][4];
            unsigned codes[2][8];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int at = step * 64 + s * 32 + 8 * g;
                f.bits[s] = pm ? pm[min(at, n - 1) >> 3] : 255u;
                k8_eight_rows(d.w, d.ldw, d.n, d.k, at, k0 + 4 * c, codes[s]);
            }
            if (step * 64 + 64 <= n) {
#pragma unroll
                for (int s = 0; s < 2; s++) { f.x[s].load(px + step * 64 + s * 32 + 8 * g); f.sw[s].load(d.sw + step * 64 + s * 32 + 8 * g); }
            } else {
#pragma unroll
                for (int s = 0; s < 2; s++) { const int at = step * 64 + s * 32 + 8 * g; f.x[s].load(px + at, n - at); f.sw[s].load(d.sw + at, n - at); }
            }
            f.pieces(true);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                k8_columns(codes[s], b[s]);
#pragma unroll
                for (int t = 0; t < 4; t++) b[s][t] = k8_bf16_codes(b[s][t]);
            }
            f.add(b, sum);
        }
    };
    for (int64_t u = u0; u < u1; u += K8_MARKS) {
        const int marked = k8_marks(a.dx + u, u1 - u, lst, before);
        k8_f32x4 sum[4];
        if (a.rows == 16)                                  // few output channels: a wavefront takes a mark's rows by itself
            for (int i = wave; i < marked; i += 8) {
                const int64_t first = (u + k8_uniform(lst[i])) * 16;
                product(min(first + c, d.m - 1), 0, 1, sum);
#pragma unroll
                for (int q = 0; q < 4; q++)                // D: column lane & 15, row 4 g + q
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        if (first + 4 * g + q < d.m && k0 + 4 * c + t < d.k) ((T *)d.dx)[(first + 4 * g + q) * d.ldx + k0 + 4 * c + t] = (T)sum[t][q];
            }
        else
            for (int i0 = 0; i0 < marked; i0 += 16) {
                const int m = min(marked - i0, 16);
                product(u + lst[i0 + min(c, m - 1)], wave, 8, sum);
                k8_few_join(sums, sum, m, (int)min((int64_t)64, d.k - k0), [&](int r, int kk, float v) __attribute__((always_inline)) {
                    ((T *)d.dx)[(u + lst[i0 + r]) * d.ldx + k0 + kk] = (T)v;
                });
                __syncthreads();                           // the sums are read
            }
        __syncthreads();                                   // the places are read
    }
}
template <class T>
__device__ __forceinline__ void k8_dw_again(const dn_i8_grad_desc &d, const K8Again &a, unsigned block, char *lds, int *lst, int *before) {
    const int tid = threadIdx.x, lane = tid & 63, wave = k8_uniform(tid >> 6), c = lane & 15, g = lane >> 4;
    const int64_t z = block / (a.blocks_k * a.blocks_n), bn = block / a.blocks_k % a.blocks_n, n0 = bn * 64, k0 = (int64_t)(block % a.blocks_k) * 256;
    const int64_t t0 = z * (a.o.run / a.rt), t1 = min((z + 1) * (a.o.run / a.rt), a.o.row_tiles);
    const uint8_t *marks = a.o.again + bn * a.o.row_tiles;
    const int nt = wave >> 1, kt = (wave & 1) * 8;         // what a wavefront multiplies: 16 output channels, 128 input channels
    const int ncols = (int)min((int64_t)64, d.n - n0);
    // a channel's 64 rows: 128 bytes; its pieces of 16 bytes lie where sixteen channels' reach different banks
    auto place = [&](int channel, int piece) { return channel * 128 + ((piece ^ (channel >> 1 & 7)) << 4); };
    char *lq = lds + 3 * 8192;
    bool any = false;
    k8_f32x4 acc[8];
#pragma unroll
    for (int t = 0; t < 8; t++) acc[t] = k8_f32x4{ 0, 0, 0, 0 };
    for (int64_t u = t0; u < t1; u += K8_MARKS) {
        const int marked = k8_marks(marks + u, t1 - u, lst, before);
        any |= marked > 0;
        for (int i = 0; i < marked; i++) {
            const int64_t first = (u + lst[i]) * a.rt, end = min(first + a.rt, d.m);
            for (int64_t r0 = first; r0 < end; r0 += 64) {
                const int rows = (int)min((int64_t)64, end - r0);
                // a thread's tasks: eight rows of one output channel and of four input channels.  A step's numbers are asked for all at once; those behind the
                // rows and the channels repeat the last ones and count as zeros (input channels: are not stored).  Little code: it is run by few, and fetched for each
                const int ch = min(lane, ncols - 1);
                T raw[8];
                float s[8];
                unsigned bit[8], codes[8];
                k8_eight_rows(d.q, d.ldq, end, d.k, r0 + wave * 8, k0 + 4 * lane, codes);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int64_t r = r0 + min(wave * 8 + e, rows - 1);
                    raw[e] = ((const T *)d.dy)[r * d.ldy + n0 + ch];
                    s[e] = d.s[r];
                    bit[e] = 255u;
                }
                if (d.mask)                                // (one branch: a load in a branch of its own is waited for there)
#pragma unroll
                    for (int e = 0; e < 8; e++) bit[e] = d.mask[(r0 + min(wave * 8 + e, rows - 1)) * d.ldmask + ((n0 + ch) >> 3)];
                __syncthreads();                           // the last step's operands are read
                i32x4 o[3];
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    float v[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int e = 2 * p + h;
                        const bool in = wave * 8 + e < rows && lane < ncols;
                        v[h] = (in && (bit[e] >> (ch & 7) & 1u) ? (float)raw[e] : 0.0f) * (in ? s[e] : 0.0f);
                    }
#pragma unroll
                    for (int i = 0; i < 3; i++) o[i][p] = k8_bf16_take(v[0], v[1]);
                }
#pragma unroll
                for (int i = 0; i < 3; i++) *(i32x4 *)(lds + i * 8192 + place(lane, wave)) = o[i];
                i32x4 q[4];
                k8_columns(codes, q);
#pragma unroll
                for (int j = 0; j < 4; j++) *(i32x4 *)(lq + place(4 * lane + j, wave)) = k8_bf16_codes(q[j]);
                __syncthreads();
                for (int p = a.pieces - 1; p >= 0; p--)    // the small ones first
#pragma unroll
                    for (int step = 0; step < 2; step++) {
                        const i32x4 u = *(const i32x4 *)(lds + p * 8192 + place(nt * 16 + c, step * 4 + g));
#pragma unroll
                        for (int t = 0; t < 8; t++) acc[t] = k8_mfma16b(u, *(const i32x4 *)(lq + place((kt + t) * 16 + c, step * 4 + g)), acc[t]);
                    }
            }
        }
    }
    if (!any) return;
    // D: column lane & 15, row 4 g + i.  The run's results are all asked for before the first is written
    const int64_t nn = n0 + nt * 16 + 4 * g, kk = k0 + kt * 16 + c;
    float *part = a.o.part + (z * d.n + nn) * d.k + kk;
    float run[8][4];
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) run[t][i] = part[min((int64_t)i, d.n - 1 - nn) * d.k + min((int64_t)t * 16, d.k - 1 - kk)];
    auto put = [&](auto *to, int64_t pitch) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 8; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (nn + i < d.n && kk + t * 16 < d.k) to[(nn + i) * pitch + kk + t * 16] = (std::remove_pointer_t<decltype(to)>)(run[t][i] + acc[t][i]);
    };
    if (a.o.splits > 1) put(a.o.part + z * d.n * d.k, d.k);
    else if (d.dw_type == DN_T_F32) put((float *)d.dw, d.lddw);
    else if (d.dw_type == DN_T_F16) put((_Float16 *)d.dw, d.lddw);
    else put((k8_bf16 *)d.dw, d.lddw);
}
template <class T>
__global__ __launch_bounds__(512) void k8_again(dn_i8_grad_desc d, K8Again a) {
    __shared__ __align__(16) char lds[7 * 8192];
    __shared__ int lst[K8_MARKS], before[8];
    if (blockIdx.x < a.dx_blocks) { k8_dx_again<T>(d, a, *(float (*)[8][4][256])lds, lst, before); return; }
    // eight of the results' blocks are looked at together, a wavefront each
    const unsigned all = (unsigned)a.o.splits * a.blocks_n * a.blocks_k, stride = gridDim.x - a.dx_blocks, wave = k8_uniform(threadIdx.x >> 6);
    for (unsigned b = blockIdx.x - a.dx_blocks; b < all; b += 8 * stride) {
        const unsigned mine = b + wave * stride;
        bool set = false;
        if (mine < all) {
            const int64_t z = mine / (a.blocks_k * a.blocks_n), t0 = z * (a.o.run / a.rt), t1 = min((z + 1) * (a.o.run / a.rt), a.o.row_tiles);
            for (int64_t t = t0 + (threadIdx.x & 63); t < t1; t += 64) set |= a.o.again[mine / a.blocks_k % a.blocks_n * a.o.row_tiles + t] != 0;
        }
        set = __any(set);
        if ((threadIdx.x & 63) == 0) lst[wave] = set;
        __syncthreads();
        unsigned marked = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) marked |= (lst[w] ? 1u : 0u) << w;
        marked = k8_uniform(marked);
        __syncthreads();
        for (int w = 0; w < 8; w++)
            if (marked >> w & 1) k8_dw_again<T>(d, a, b + w * stride, lds, lst, before);
    }
}

// ---- dw and db, few rows (M <= 16) ------------------------------------------------------------------------------------------------------------------------------
// dw's bytes are all there is to move.  The factors dz s and the codes go as they are, in fp32, into matrix instructions over four rows; 64 x 64 results per wavefront,
// tile t of a block holds input channels 4 c + t, so that a lane stores four adjacent ones.  No LDS, no waiting for one another.
// 6 x 1991 x 3807 fp16 10 us (k8_dw: 24), 12 x 4096 x 4096 bf16 19 us for 34 MB (k8_dw: 20; as fp32 vector products: 22).
template <class T, class W>
__global__ __launch_bounds__(256) void k8_dw_few(dn_i8_grad_desc d) {
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4, m = (int)d.m;
    const int64_t n0 = (int64_t)blockIdx.y * 64, k0 = (int64_t)blockIdx.x * 256 + wave * 64, left = d.k - k0 - 4 * c;
    const bool with_q = d.dw && k0 < d.k;
    float u[4][4], sum[4] = { 0, 0, 0, 0 }, scale[4] = { 0, 0, 0, 0 };
    unsigned q[4] = { 0, 0, 0, 0 };
    int64_t row[4], col[4];                                // rows 4 s + g; those behind the last one repeat it and count as zeros
#pragma unroll
    for (int s = 0; s < 4; s++) { row[s] = min(4 * s + g, m - 1); col[s] = min(n0 + 16 * s + c, d.n - 1); }
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
        for (int b = 0; b < 4; b++) u[b][s] = (float)((const T *)d.dy)[row[s] * d.ldy + col[b]];
    if (with_q) {
#pragma unroll
        for (int s = 0; s < 4; s++) scale[s] = d.s[row[s]];
        const int8_t *p = d.q + k0 + 4 * c;
        if (k0 + 64 <= d.k)
#pragma unroll
            for (int s = 0; s < 4; s++) __builtin_memcpy(&q[s], p + row[s] * d.ldq, 4);
        else
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int j = 0; j < 4; j++) q[s] |= (unsigned)(uint8_t)p[row[s] * d.ldq + min((int64_t)j, left - 1)] << (8 * j);        // the row's last code stands for those behind it
    }
    if (d.mask) {
        unsigned bits[4][4];
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int b = 0; b < 4; b++) bits[b][s] = d.mask[row[s] * d.ldmask + (col[b] >> 3)];
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int b = 0; b < 4; b++) u[b][s] = bits[b][s] >> (col[b] & 7) & 1 ? u[b][s] : 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const float z = 4 * s + g < m ? u[b][s] : 0.0f;
            sum[b] += z;
            u[b][s] = 4 * s + g < m ? z * scale[s] : 0.0f;
        }
    if (with_q)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            k8_f32x4 acc[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                acc[t] = k8_f32x4{ 0, 0, 0, 0 };
#pragma unroll
                for (int s = 0; s < 4; s++)
                    if (4 * s < m) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[b][s], (float)(int8_t)(q[s] >> (8 * t)), acc[t], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t n = n0 + 16 * b + 4 * g + i;
                const float v[4] = { acc[0][i], acc[1][i], acc[2][i], acc[3][i] };
                if (n < d.n && left > 0) k8_put4((W *)d.dw + n * d.lddw + k0 + 4 * c, v, left);
            }
        }
    if (d.db && blockIdx.x == 0 && wave == 0)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            sum[b] += __shfl_xor(sum[b], 16);
            sum[b] += __shfl_xor(sum[b], 32);
            const int64_t n = n0 + 16 * b + c;
            if (g == 0 && n < d.n) k8_put1(d.db, d.dw_type, n, sum[b]);
        }
}

// few runs joined: a lane takes four adjacent results of all of them
__global__ __launch_bounds__(256) void k8_dw_join_few(const float *__restrict__ part, const float *__restrict__ part_b, int splits, int64_t n, int64_t k, void *__restrict__ dw,
                                                      int64_t lddw, void *__restrict__ db, int type, unsigned dw_blocks) {
    const bool is_b = blockIdx.x >= dw_blocks;
    const int64_t count = is_b ? n : n * k, at = ((int64_t)(is_b ? blockIdx.x - dw_blocks : blockIdx.x) * 256 + threadIdx.x) * 4, left = count - at;
    if (left <= 0) return;
    const float *p = (is_b ? part_b : part) + at;
    float v[4] = { 0, 0, 0, 0 };
    if (left >= 4)
#pragma unroll 8
        for (int z = 0; z < splits; z++) {
            const K8Vec<float, 4> t = k8_load<float, 4>(p + (int64_t)z * count);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += t.v[j];
        }
    else
        for (int z = 0; z < splits; z++)
#pragma unroll
            for (int j = 0; j < 3; j++) if (j < left) v[j] += p[(int64_t)z * count + j];
    void *out = is_b ? db : dw;
    const int64_t r = is_b ? 0 : at / k, c = is_b ? at : at - r * k;
    if (left >= 4 && (is_b || c + 4 <= k)) { k8_put4(out, type, is_b ? at : r * lddw + c, v, 4); return; }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (j < left) {
            const int64_t o = is_b ? at + j : (at + j) / k * lddw + (at + j) % k;
            if (type == DN_T_F32) ((float *)out)[o] = v[j];
            else if (type == DN_T_F16) ((_Float16 *)out)[o] = (_Float16)v[j];
            else ((k8_bf16 *)out)[o] = (k8_bf16)v[j];
        }
}
// the runs joined, dw's and db's in one launch.  A workgroup takes 256 adjacent results: 64 lanes x four, 16 wavefronts a sixteenth of the runs each, so that a
// run's loads are all in flight at once
__global__ __launch_bounds__(1024) void k8_dw_join(const float *__restrict__ part, const float *__restrict__ part_b, int splits, int64_t n, int64_t k, void *__restrict__ dw,
                                                   int64_t lddw, void *__restrict__ db, int type, unsigned dw_blocks) {
    __shared__ float js[16][256];
    const bool is_b = blockIdx.x >= dw_blocks;
    const int64_t count = is_b ? n : n * k, at = (int64_t)(is_b ? blockIdx.x - dw_blocks : blockIdx.x) * 256;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t mine = at + lane * 4, left = count - mine;
    float v[4] = { 0, 0, 0, 0 };
    if (left > 0) {
        const float *p = (is_b ? part_b : part) + mine;
        for (int z0 = wave; z0 < splits; z0 += 256) {      // sixteen runs a wavefront, all of them asked for before the first is added
            K8Vec<float, 4> t[16];
#pragma unroll
            for (int u = 0; u < 16; u++) {
                const float *q = p + (int64_t)min(z0 + 16 * u, splits - 1) * count;
                if (left >= 4) t[u] = k8_load<float, 4>(q);
                else
#pragma unroll
                    for (int j = 0; j < 4; j++) t[u].v[j] = j < left ? q[j] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 16; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] += z0 + 16 * u < splits ? t[u].v[j] : 0.0f;
        }
    }
    *(k8_f32x4 *)(&js[wave][lane * 4]) = k8_f32x4{ v[0], v[1], v[2], v[3] };
    __syncthreads();
    const int64_t o = at + threadIdx.x;
    if (threadIdx.x >= 256 || o >= count) return;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) s += js[w][threadIdx.x];
    const int64_t to = is_b ? o : o / k * lddw + o % k;
    void *out = is_b ? db : dw;
    if (type == DN_T_F32) ((float *)out)[to] = s;
    else if (type == DN_T_F16) ((_Float16 *)out)[to] = (_Float16)s;
    else ((k8_bf16 *)out)[to] = (k8_bf16)s;
}

// ---- which way a call takes.  Nothing here looks at which results are asked for: a result's bits do not depend on its company -----------------------------------------
struct Plan {
    bool few = false, narrow = false; K8Tiling tile = K8_BIG; int dx_splits = 1, np_x = 1, np_w = 1, pitch = 0;
    int s = 256, rt = 64, tiles_n = 1, tiles_k = 1, splits = 1; int64_t run = 0, row_tiles = 1;
    uint64_t pieces = 0, turned = 0, down = 0, dx_part = 0, dx_again = 0, dw_again = 0, part = 0, part_b = 0, total = 0;
};
Plan plan_grad(const dn_i8_grad_desc &d) {
    Plan p;
    auto take = [&](uint64_t bytes) { const uint64_t at = p.total; p.total += k8_up(bytes, 256); return at; };
    p.np_x = d.dy_type == DN_T_F32 ? 2 : 1;
    p.np_w = d.dw_type == DN_T_F32 ? 2 : 1;
    // us, dx and dw, bf16, few : tiles -- 16 x 1024 x 1024, 14 : 27; 16 x 4096 x 4096, 32 : 55; 1 x 64 x 64, 9 : 18
    p.few = d.m >= 1 && d.m <= 16 && d.k >= 4;
    // one launch that reads dy once for 256 input channels, behind a weight that every workgroup lays out first.  us, dx and dw, bf16, this : pieces and tiles (M x K x N) --
    // 8000 x 64 x 64, 21 : 29; 100 x 1024 x 128, 21 : 23; 5000 x 4096 x 64, 43 : 61; 300 x 256 x 256, 31 : 26; 2000 x 1024 x 256, 41 : 37; 50000 x 256 x 256, 67 : 83;
    // 50000 x 2048 x 200, 184 : 264
    p.narrow = d.k <= 4096 && (d.n <= 128 || (d.n <= 256 && d.m * ((d.k + 255) / 256) >= 16384));
    if (p.few) {
        p.dx_splits = (int)std::max<int64_t>(1, std::min<int64_t>(K8_CUS / ((d.k + 63) / 64), d.n / 1024));
        if (d.dx && p.dx_splits > 1) p.dx_part = take((uint64_t)p.dx_splits * d.m * d.k * 4);
        return p;
    }
    if (d.dx && d.m && !p.narrow) {
        p.pitch = (int)k8_up(d.n, 8);
        p.pieces = take((uint64_t)p.np_x * d.m * p.pitch * 2);
        p.turned = take((uint64_t)d.k * p.pitch * 2);
        p.down = take((uint64_t)d.m * 4);
        p.tile = k8_tiling(d.m, d.k);
        const int64_t tiles = k8_tiles(p.tile, d.m, d.k), steps = (p.pitch * 2 + 127) / 128 * p.np_x;
        if (tiles < K8_CUS) {
            p.dx_splits = (int)std::max<int64_t>(1, std::min<int64_t>(K8_CUS / tiles, steps / 4));
            if (p.dx_splits > 1) p.dx_part = take((uint64_t)p.dx_splits * d.m * d.k * 4);
        }
    }
    if (d.dx && d.m) p.dx_again = take(p.narrow ? (uint64_t)(d.m + 15) / 16 : (uint64_t)d.m);
    int64_t want = K8_CUS;
    // dw's tiles and the runs of rows: what costs least, by times measured on whole chips -- a workgroup's row in a tile of 256: 55 ns (fp16, fp32: 65), of 128: 21; its start and
    // end: 14 us and 9; a run's results, written and read again: 1.2 ps each.  bf16, us, 256 : 128 -- 1048576 x 256 x 256, 281 : 345; 200000 x 192 x 192, 73 : 89;
    // 50000 x 1024 x 256, 103 : 85; 7552 x 1664 x 1216, 82 : 139; 1000 x 1024 x 1024, 39 : 23; 64 x 2048 x 4096, 20 : 26;
    // with dx, fp16, 12824 x 1088 x 2304, 310 : 338; fp32, 100000 x 256 x 256, 131 : 116.  (Of a lane's 256 registers tiles of 256 lack 5 for bf16 and 7 for fp16; for fp32 17,
    // or 80 with fp32 results: those go to memory.)
    if (std::max(d.n, d.k) <= 64) p.s = 64;
    else {
        double least = 1e30;
        for (int side : { 128, 256 }) {
            const int64_t tiles = ((d.n + side - 1) / side) * ((d.k + side - 1) / side), most = std::max<int64_t>(1, (d.m * p.np_w * side + 16383) / 16384);
            for (int rounds = 1; rounds <= 3; rounds++) {
                const int64_t runs = std::min(most, std::max<int64_t>(1, rounds * K8_CUS / tiles)), turns = (tiles * runs + K8_CUS - 1) / K8_CUS;
                const double cost = (double)turns * ((side == 256 ? 14e3 : 9e3) + (side == 256 ? (d.dy_type == DN_T_BF16 ? 55.0 : 65.0) : 21.0) * (double)(d.m * p.np_w) / (double)runs) +
                                    (runs > 1 ? 3e3 + 1.2e-3 * (double)(runs * d.n * d.k) : 0.0);
                if (cost < least) { least = cost; p.s = side; want = runs; }
            }
        }
    }
    const int64_t rt = 16384 / p.s / p.np_w, row_tiles = std::max<int64_t>(1, (d.m + rt - 1) / rt);
    p.tiles_n = (int)((d.n + p.s - 1) / p.s); p.tiles_k = (int)((d.k + p.s - 1) / p.s);
    const int64_t each = (row_tiles + want - 1) / want;
    p.run = each * rt;
    p.splits = (int)((row_tiles + each - 1) / each);
    p.row_tiles = row_tiles; p.rt = (int)rt;
    if (d.dw) {
        p.part = take((uint64_t)p.splits * d.n * d.k * 4);
        p.dw_again = take((uint64_t)p.tiles_n * (p.s / 64) * row_tiles);
    }
    if (p.splits > 1) {
        if (d.db) p.part_b = take((uint64_t)p.splits * d.n * 4);
    }
    return p;
}

template <class T, int NP, class Epi> hipError_t dx_gemm(const dn_i8_grad_desc &d, const Plan &p, char *base, const Epi &e, hipStream_t st) {
    const int64_t plane = d.m * (int64_t)p.pitch * 2;
    return k8_product<false>(G8{ base + p.pieces, base + p.turned, (int64_t)p.pitch * 2, (int64_t)p.pitch * 2, d.m, d.k, p.pitch * 2, NP, plane, p.dx_splits, 0, 0 }, p.tile, e, st);
}
template <class T, int NP> hipError_t dx_of(const dn_i8_grad_desc &d, const Plan &p, char *base, hipStream_t st) {
    if (p.few) {
        const int run = (int)k8_up((d.n + p.dx_splits - 1) / p.dx_splits, 64);
        float *part = p.dx_splits > 1 ? (float *)(base + p.dx_part) : nullptr;
        k8_dx_few<T><<<dim3((unsigned)((d.k + 63) / 64), (unsigned)p.dx_splits), 512, 0, st>>>(d, run, part);
        if (part) k8_dx_join<T><<<dim3((unsigned)((d.m * ((d.k + 255) / 256) + 3) / 4)), 256, 0, st>>>(part, p.dx_splits, nullptr, (T *)d.dx, d.m, d.k, d.ldx);
        return hipGetLastError();
    }
    uint8_t *again = (uint8_t *)base + p.dx_again;
    if (p.narrow) {
        const unsigned per = (unsigned)((d.k + 255) / 256);
        auto grid = [&](int each) { return dim3((unsigned)std::min<int64_t>((d.m + 127) / 128, each * K8_CUS / per), per); };      // a wavefront has 16 rows
        if (d.n <= 64) k8_dx_narrow<T, 2, NP><<<grid(4), 512, 0, st>>>(d, again);
        else if (d.n <= 128) k8_dx_narrow<T, 4, NP><<<grid(2), 512, 0, st>>>(d, again);
        else k8_dx_narrow<T, 8, NP><<<grid(1), 512, 0, st>>>(d, again);
        return hipGetLastError();
    }
    _Float16 *pieces = (_Float16 *)(base + p.pieces), *turned = (_Float16 *)(base + p.turned);
    float *down = (float *)(base + p.down);
    const int64_t plane = d.m * (int64_t)p.pitch;
    for (int64_t r = 0; r < d.m; r += K8_LAUNCH_ROWS) {
        dn_i8_grad_desc t = d;
        t.m = std::min(d.m - r, K8_LAUNCH_ROWS);
        t.dy = (const T *)d.dy + r * d.ldy;
        if (d.mask) t.mask = d.mask + r * d.ldmask;
#define PIECES(LPR_, V_) k8_pieces<T, LPR_, V_, NP><<<dim3((unsigned)((t.m + 256 / LPR_ - 1) / (256 / LPR_))), 256, 0, st>>>(t, pieces + r * p.pitch, p.pitch, plane, down + r, again + r)
        if (d.n <= 512) PIECES(64, 1);
        else if (d.n <= 1024) PIECES(64, 2);
        else if (d.n <= 2048) PIECES(64, 4);
        else if (d.n <= 4096) PIECES(256, 2);
        else if (d.n <= 8192) PIECES(256, 4);
        else PIECES(256, 0);
#undef PIECES
    }
    k8_turn<<<dim3((unsigned)(((p.pitch + 63) / 64) * ((d.k + 127) / 128))), 256, 0, st>>>(d, turned, p.pitch);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.dx_splits == 1) return dx_gemm<T, NP>(d, p, base, DxEpi<T>{ down, (T *)d.dx, d.k, d.ldx }, st);
    const DxPart part = { (float *)(base + p.dx_part), d.m, d.k };
    e = dx_gemm<T, NP>(d, p, base, part, st);
    if (e != hipSuccess) return e;
    k8_dx_join<T><<<dim3((unsigned)((d.m * ((d.k + 255) / 256) + 3) / 4)), 256, 0, st>>>(part.part, p.dx_splits, down, (T *)d.dx, d.m, d.k, d.ldx);
    return hipGetLastError();
}
template <class T, int NP> hipError_t dw_of(const dn_i8_grad_desc &d, const Plan &p, char *base, hipStream_t st) {
    if (p.few) {
        const dim3 grid(d.dw ? (unsigned)((d.k + 255) / 256) : 1u, (unsigned)((d.n + 63) / 64));
        if (d.dw_type == DN_T_F32) k8_dw_few<T, float><<<grid, 256, 0, st>>>(d);
        else if (d.dw_type == DN_T_F16) k8_dw_few<T, _Float16><<<grid, 256, 0, st>>>(d);
        else k8_dw_few<T, k8_bf16><<<grid, 256, 0, st>>>(d);
        return hipGetLastError();
    }
    const int tiles_k = d.dw ? p.tiles_k : 1;
    const DwOut o = { (float *)(base + p.part), (float *)(base + p.part_b), p.splits, p.tiles_n, tiles_k, p.run, (uint8_t *)base + p.dw_again, p.row_tiles };
    const dim3 grid((unsigned)((int64_t)p.splits * p.tiles_n * tiles_k));
    if (p.s == 64) k8_dw<T, 64, NP><<<grid, 512, 0, st>>>(d, o);
    else if (p.s == 128) k8_dw<T, 128, NP><<<grid, 512, 0, st>>>(d, o);
    else k8_dw<T, 256, NP><<<grid, 512, 0, st>>>(d, o);
    return hipGetLastError();
}
// what is marked, then dw's runs joined
template <class T> hipError_t finish(const dn_i8_grad_desc &d, const Plan &p, char *base, hipStream_t st) {
    if (p.few || !d.m) return hipSuccess;
    K8Again a = {};
    if (d.dx) {
        a.dx = (const uint8_t *)base + p.dx_again; a.rows = p.narrow ? 16 : 1; a.units = p.narrow ? (d.m + 15) / 16 : d.m;
        a.cols = (unsigned)((d.k + 63) / 64);
        a.slices = (unsigned)std::min<int64_t>((a.units + 63) / 64, std::max<int64_t>(1, K8_CUS / a.cols));
        a.dx_blocks = a.cols * a.slices;
    }
    a.o = { (float *)(base + p.part), (float *)(base + p.part_b), p.splits, p.tiles_n, p.tiles_k, p.run, (uint8_t *)base + p.dw_again, p.row_tiles };
    unsigned dw_blocks = 0;
    if (d.dw) {
        a.rt = p.rt; a.pieces = p.np_w + 1;
        a.blocks_n = (unsigned)((d.n + 63) / 64); a.blocks_k = (unsigned)((d.k + 255) / 256);
        dw_blocks = (unsigned)std::min<int64_t>((int64_t)p.splits * a.blocks_n * a.blocks_k, 2 * K8_CUS);
    }
    if (a.dx_blocks + dw_blocks) k8_again<T><<<dim3(a.dx_blocks + dw_blocks), 512, 0, st>>>(d, a);
    const DwOut &o = a.o;
    if (p.splits > 1 && (d.dw || d.db)) {
        // many runs of few results: their loads shared by sixteen wavefronts (200000 x 64 x 64, 44.1 us: 47.0 without), else four results of all runs per lane
        // (5000 x 256 x 256, 34 us: 43 the other way; 7552 x 1664 x 1216, 82: 169)
        const int64_t each = p.splits > 8 && d.n * d.k < 128 * K8_CUS ? 256 : 1024;
        const unsigned dw_blocks = d.dw ? (unsigned)((d.n * d.k + each - 1) / each) : 0, db_blocks = d.db ? (unsigned)((d.n + each - 1) / each) : 0;
        if (each == 1024) k8_dw_join_few<<<dim3(dw_blocks + db_blocks), 256, 0, st>>>(o.part, o.part_b, p.splits, d.n, d.k, d.dw, d.lddw, d.db, d.dw_type, dw_blocks);
        else k8_dw_join<<<dim3(dw_blocks + db_blocks), 1024, 0, st>>>(o.part, o.part_b, p.splits, d.n, d.k, d.dw, d.lddw, d.db, d.dw_type, dw_blocks);
    }
    return hipGetLastError();
}

}  // namespace

uint64_t k8_grad_workspace(const dn_i8_grad_desc &d) { return plan_grad(d).total; }

template <class T> static hipError_t grad_of(const dn_i8_grad_desc &d, const Plan &p, char *base, hipStream_t st) {
    hipError_t e = hipSuccess;
    if (d.dx && d.m) e = dx_of<T, sizeof(T) / 2>(d, p, base, st);
    if (e == hipSuccess && (d.dw || d.db)) e = p.np_w == 2 ? dw_of<T, 2>(d, p, base, st) : dw_of<T, 1>(d, p, base, st);
    if (e == hipSuccess) e = finish<T>(d, p, base, st);
    return e;
}
hipError_t k8_grad(const dn_i8_grad_desc &d, void *ws, hipStream_t st) {
    const Plan p = plan_grad(d);
    switch (d.dy_type) {
        case DN_T_F32: return grad_of<float>(d, p, (char *)ws, st);
        case DN_T_F16: return grad_of<_Float16>(d, p, (char *)ws, st);
        default: return grad_of<k8_bf16>(d, p, (char *)ws, st);
    }
}
