// k8_gemm.h -- the matrix product under the 8-bit dense layers: C = A B^T for rows of 8-bit integers (32-bit integer sums) or of fp16 numbers (fp32
// sums).  Both operands have the reduction along their rows, so an operand row is a run of bytes whatever its type: 16 bytes are what one lane feeds a
// matrix instruction (16 integers or 8 fp16), 128 bytes per row and step go through LDS, and one kernel serves both.
//
//   tile      BM x BN results per workgroup, WGM x WGN wavefronts, each (BM / WGM) x (BN / WGN) results in 32 x 32 blocks
//   loads     buffer loads straight into LDS, 16 bytes per lane, two stages; the next step's loads are in flight while this one multiplies.  Rows behind
//             the matrix and bytes behind the row's end read as zeros (bounds of the buffer descriptor; an offset no buffer has)
//   LDS       a row's eight 16-byte pieces are stored at piece ^ (row / 2 & 7): sixteen neighbouring lanes of an operand read (sixteen rows, two to a line of the 64
//             banks) hit sixteen different places
//   results   block t of a wavefront holds columns TN c + t (c = lane & 31): a lane's TN blocks are adjacent columns, and a row leaves in runs of
//             32 TN columns instead of 32
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float k8_f32x4 __attribute__((ext_vector_type(4)));
typedef float k8_f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 k8_f16x8 __attribute__((ext_vector_type(8)));

struct G8 {
    const char *a, *b;           // rows at pitches of lda, ldb BYTES (multiples of 16, like the addresses)
    int64_t lda, ldb;
    int64_t m, n;                // rows of a, rows of b
    int kb;                      // bytes of a row that count; i8: any number, fp16: a multiple of 16 (zeros behind the numbers)
    int planes;                  // the reduction runs over planes of a (plane_a bytes apart) against the same b; two (fp16): the first one's sums count 2^-12
    int64_t plane_a;
    int splits;                  // the reduction is cut into that many runs of steps; run z of a tile is result z
    int tiles_m, tiles_n;
};

template <bool I8> struct K8Acc { typedef i32x16 type; };
template <> struct K8Acc<false> { typedef k8_f32x16 type; };

__device__ __forceinline__ i32x16 k8_mfma32(i32x4 a, i32x4 b, i32x16 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ k8_f32x16 k8_mfma32(i32x4 a, i32x4 b, k8_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(k8_f16x8, a), __builtin_bit_cast(k8_f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ int k8_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const char *k8_uniform(const char *p) {
    const uint64_t v = (uint64_t)p;
    return (const char *)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

// global memory behind a uniform address: one 32-bit offset per lane does, and the loads are global ones (a pointer made from integers alone is a generic one)
typedef const __attribute__((address_space(1))) char *k8_global;
__device__ __forceinline__ k8_global k8_base(const void *p) { return (k8_global)k8_uniform((const char *)p); }

// which tile a workgroup takes.  Workgroups are dealt to the eight XCDs round-robin: XCD x takes a contiguous run of tiles, and inside the run tiles go
// column block by column block over groups of eight row blocks, so that what an XCD works on at a time shares rows of a and of b in its own L2
struct K8Tile { int tm, tn, z; };
__device__ __forceinline__ K8Tile k8_tile(const G8 &g, int bid, int total) {
    const int per = total >> 3, rest = total & 7, x = bid & 7, i = bid >> 3;
    const int id = x * per + min(x, rest) + i;             // XCD x has per (+ 1 if x < rest) workgroups
    const int tiles = g.tiles_m * g.tiles_n, z = id / tiles, t = id - z * tiles;
    const int group = 8 * g.tiles_n, gi = t / group, first = gi * 8, size = min(8, g.tiles_m - first), r = t - gi * group;
    return { first + r % size, r / size, z };
}

// The epilogue: columns(a lane's first column), row(row, column), store(those, row, column, run z, values of TN adjacent columns, whether the row and column exist)
template <bool I8, int BM, int BN, int WGM, int WGN, class Epi>
__global__ __launch_bounds__(64 * WGM * WGN) void k8_gemm(G8 g, Epi epi) {
    constexpr int NW = WGM * WGN, TM = BM / WGM / 32, TN = BN / WGN / 32, LOADS = (BM + BN) / 8 / NW;
    static_assert((BM + BN) % (8 * NW) == 0 && BM % (8 * NW) == 0, "whole loads per wavefront, each of one operand");
    __shared__ __align__(1024) char l0[(BM + BN) * 128];
    __shared__ __align__(1024) char l1[(BM + BN) * 128];
    typedef typename K8Acc<I8>::type acc_t;
    const int lane = threadIdx.x & 63, wave = k8_uniform(threadIdx.x >> 6), wm = wave / WGN, wn = wave % WGN;
    const K8Tile t = k8_tile(g, blockIdx.x, gridDim.x);
    const int64_t m0 = (int64_t)t.tm * BM, n0 = (int64_t)t.tn * BN;
    const int rows_a = (int)min((int64_t)BM, g.m - m0), rows_b = (int)min((int64_t)BN, g.n - n0);
    // bytes of a tile's rows that may be read: whole 16-byte pieces up to the one with the last row's last counted byte (it cannot cross a page)
    const unsigned na = (unsigned)((int64_t)(rows_a - 1) * g.lda + ((g.kb + 15) & ~15)), nb = (unsigned)((int64_t)(rows_b - 1) * g.ldb + ((g.kb + 15) & ~15));
    const char *pa = k8_uniform(g.a + m0 * g.lda), *pb = k8_uniform(g.b + n0 * g.ldb);
    const int per_plane = (g.kb + 127) >> 7, steps = per_plane * g.planes;
    const int s0 = (int)((int64_t)steps * t.z / g.splits), s1 = (int)((int64_t)steps * (t.z + 1) / g.splits);
    // Load i of a wavefront covers rows 8 (i NW + wave) .. + 7 of the stage, first a's, then b's; a stage row of b in a block of 64 holds the block's matrix row
    // 2 c + t at 32 t + c (what a wavefront reads for its block t is then 32 rows in a row).  The lane's row and piece are the same in every load of an operand: only
    // the buffer's base moves, and with it how many bytes of the tile are left
    static_assert(TN == 2 && (NW == 4 || NW == 8), "how b's rows are dealt to the loads");
    const int row8 = wave * 8 + (lane >> 3);
    const int piece = ((lane & 7) ^ ((row8 >> 1) & 7)) * 16;
    const unsigned off_a = (unsigned)(row8 * g.lda) + piece, off_b = (unsigned)(((row8 & 31) * 2 + (row8 >> 5)) * g.ldb) + piece;
    auto fetch = [&](char *l, int s, int from, int to) __attribute__((always_inline)) {        // loads from .. to - 1 of step s
        const int plane = s / per_plane, k = (s - plane * per_plane) << 7;
        const bool any = s >= s0;
        const bool in = any && k + piece < g.kb;
        const unsigned oa = in ? off_a + (unsigned)k : 0x80000000u, ob = in ? off_b + (unsigned)k : 0x80000000u;
        const char *at = k8_uniform(pa + plane * g.plane_a);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (i < from || i >= to) continue;
            const bool is_a = i * NW * 8 < BM;
            const int ib = i - BM / 8 / NW, rows = is_a ? i * NW * 8 : NW == 8 ? ib * 64 : (ib >> 1) * 64 + (ib & 1);
            const unsigned skip = (unsigned)rows * (unsigned)(is_a ? g.lda : g.ldb), have = is_a ? na : nb;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)((is_a ? at : pb) + skip), 0, have > skip ? have - skip : 0u, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(l + (i * NW + wave) * 1024), 16, is_a ? oa : ob, 0, 0, 0);
        }
    };
    acc_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int q = 0; q < 16; q++) acc[i][j][q] = 0;
    const int c = lane & 31, h = lane >> 5;
    const int abase = (wm * TM * 32 + c) * 128, bbase = (BM + wn * TN * 32 + c) * 128, key = (c >> 1) & 7;
    // LAST: the row may end inside this step.  Integers behind the end: whatever is there counts as zero in one operand, which is enough
    auto multiply = [&](const char *l, int s, auto last, auto &&next) __attribute__((always_inline)) {
        i32x4 a[2][TM], b[2][TN];                          // a quarter step's operands are read while the quarter before it multiplies
        auto operands = [&](int q) __attribute__((always_inline)) {
            const int p = 2 * q + h;
#pragma unroll
            for (int i = 0; i < TM; i++) a[q & 1][i] = *(const i32x4 *)(l + abase + i * 32 * 128 + ((p ^ key) << 4));
#pragma unroll
            for (int j = 0; j < TN; j++) b[q & 1][j] = *(const i32x4 *)(l + bbase + j * 32 * 128 + ((p ^ key) << 4));
        };
        operands(0);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (q < 3) operands(q + 1);
            next(q);
            __builtin_amdgcn_sched_barrier(0);
            if (I8 && decltype(last)::value) {
                const int left = g.kb - (s << 7) - (2 * q + h) * 16;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int keep = left - 4 * e;
                    const int mask = keep >= 4 ? -1 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
#pragma unroll
                    for (int i = 0; i < TM; i++) a[q & 1][i][e] &= mask;
                }
            }
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = k8_mfma32(a[q & 1][i], b[q & 1][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // steps go in pairs, one left over goes last.  A step that cuts a row of integers has to be that one: the run then starts a step early, on zeros, if it has to
    // between the planes: what the first one summed
    auto lower = [&]() __attribute__((always_inline)) {
        if constexpr (!I8)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
#pragma unroll
                    for (int q = 0; q < 16; q++) acc[i][j][q] *= 0x1p-12f;
    };
    const int border = !I8 && g.planes == 2 ? per_plane : -1;
    const bool cut = I8 && (g.kb & 127) && s1 == steps;
    int s = s0 - (cut && !((s1 - s0) & 1) ? 1 : 0);
    // the next step's loads are asked for in the first two quarters of this one: all at once they keep the wavefronts from their products until the queue has taken
    // them (8192 x 4096 x 4096 in 8 bits: 158.5 us; two quarters 154.9; all four 157.6, the last then land late)
    constexpr int PER = LOADS / 2;
    if (s < s1) fetch(l0, s, 0, LOADS);
    for (; s + 1 < s1; s += 2) {
        __syncthreads();                                   // this step's loads have landed, and nobody reads the other stage any more
        if (!I8 && s == border) lower();
        multiply(l0, s, std::false_type(), [&](int q) __attribute__((always_inline)) { fetch(l1, s + 1, q * PER, min(q * PER + PER, LOADS)); });
        __syncthreads();
        if (!I8 && s + 1 == border) lower();
        const bool more = s + 2 < s1;
        multiply(l1, s + 1, std::false_type(), [&](int q) __attribute__((always_inline)) { if (more) fetch(l0, s + 2, q * PER, min(q * PER + PER, LOADS)); });
    }
    if (s < s1) {
        __syncthreads();
        if (!I8 && s == border) lower();
        multiply(l0, s, std::true_type(), [](int) {});
    }
    if (!I8 && s1 <= border) lower();
    // D: column lane & 31, row (q & 3) + 8 (q >> 2) + 4 h.  Lanes outside the matrix stay: an epilogue may put lanes' results together.  What it reads for 16 rows is
    // asked for before the first of them is finished
    const int64_t nn = n0 + wn * TN * 32 + c * TN;
    const auto cols = epi.template columns<TN>(nn);
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int64_t m1 = m0 + wm * TM * 32 + i * 32 + 4 * h;
        typename Epi::template Row<TN> rows[16];
#pragma unroll
        for (int q = 0; q < 16; q++) rows[q] = epi.template row<TN>(min(m1 + (q & 3) + 8 * (q >> 2), g.m - 1), nn);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < 16; q++) {
            const int64_t mm = m1 + (q & 3) + 8 * (q >> 2);
            typename Epi::value v[TN];
#pragma unroll
            for (int j = 0; j < TN; j++) v[j] = acc[i][j][q];
            epi.template store<TN>(cols, rows[q], mm, nn, t.z, v, mm < g.m && nn < g.n);
            if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);                // a few rows at a time: the registers are full
        }
    }
}

// Which tiles a product takes: 256 x 256 where that makes a tile for every compute unit, 128 x 128 where that does, 128 x 64 otherwise and where b has no more rows.
// us, the larger : the smaller tile -- 328813 x 1344 x 39 fp16, 402 (256) : 150 (64); 1500 x 2048 x 1605 bf16, 32 (128) : 25 (64); 500 x 500 x 500, 18 (128) : 12 (64);
// 200 x 4096 x 2048 of a gradient, 19 (128) : 20 (64); with the operands of 8192 x 4096 x 4096 a tile of 256 reads half as much as one of 128
enum K8Tiling { K8_BIG, K8_MIDDLE, K8_SLIM };
inline int64_t k8_tiles(K8Tiling t, int64_t m, int64_t n) {
    const int64_t bm = t == K8_BIG ? 256 : 128, bn = t == K8_BIG ? 256 : t == K8_MIDDLE ? 128 : 64;
    return ((m + bm - 1) / bm) * ((n + bn - 1) / bn);
}
inline K8Tiling k8_tiling(int64_t m, int64_t n) {
    if (n <= 64 || k8_tiles(K8_MIDDLE, m, n) < 256) return K8_SLIM;
    return k8_tiles(K8_BIG, m, n) >= 256 ? K8_BIG : K8_MIDDLE;
}
template <bool I8, class Epi> hipError_t k8_product(G8 g, K8Tiling t, const Epi &e, hipStream_t st) {
    const int bm = t == K8_BIG ? 256 : 128, bn = t == K8_BIG ? 256 : t == K8_MIDDLE ? 128 : 64;
    g.tiles_m = (int)((g.m + bm - 1) / bm); g.tiles_n = (int)((g.n + bn - 1) / bn);
    const dim3 grid((unsigned)((int64_t)g.tiles_m * g.tiles_n * g.splits));
    if (t == K8_BIG) k8_gemm<I8, 256, 256, 2, 4, Epi><<<grid, 512, 0, st>>>(g, e);
    else if (t == K8_MIDDLE) k8_gemm<I8, 128, 128, 2, 2, Epi><<<grid, 256, 0, st>>>(g, e);
    else k8_gemm<I8, 128, 64, 4, 1, Epi><<<grid, 256, 0, st>>>(g, e);
    return hipGetLastError();
}
