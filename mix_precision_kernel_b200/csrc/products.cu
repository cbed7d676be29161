// Products grouped by expert and products in 8-bit integers: persistent,
// warp-specialised tcgen05 kernels for sm_100a.
//
//   rows product      D[i] = A[i] * B[e] for the rows i of group e, which are
//                     offsets[e] <= i < offsets[e + 1]; B[e] is [K][N] or [N][K].
//                     A and B are both BF16, both FP16 or both int8; one group of all
//                     rows is the plain product.
//   weight gradient   D[e] = A[rows of e]^T * B[rows of e], a K x N matrix per group
//                     whose reduction is as long as the group.
//
// The groups' bounds are read from device memory, so that a router's result needs no
// copy to the host: every CTA scans them into shared memory (row ranges and a running
// count of tiles) and walks the tiles of all groups with a stride of the grid.
//
// Operands stream by TMA into a ring of 128-byte-wide stages (64 16-bit or 128 8-bit
// elements of the reduction), swizzled as the MMA reads them, in whatever order they
// are stored: the reduction axis may be the contiguous one (K-major) or the strided
// one (MN-major) for either operand.  A group's rows start anywhere: a load may begin
// at any row, and rows of the next group that land in a tile only make accumulator
// rows that are not stored.  Where the ragged axis is the reduction (weight gradient)
// the rows behind the group's end are zeroed in shared memory before the last MMAs.
//
// Accumulators live in tensor memory, two of them, so that a tile's epilogue runs
// under the next tile's MMAs.  FP32 sums for the 16-bit types, 32-bit integer sums
// (exact: the host refuses a K at which they could overflow) for int8.
//
// Every mbarrier wait is bounded (mpk::mbar_wait); on expiry the CTA raises an abort
// flag, records a status code, drains what it has in flight and leaves.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "mpk.h"
#include "mpk_internal.h"
#include "mpk_ptx.cuh"

namespace mpk {
namespace product {

constexpr int BM = 128;             // accumulator rows per CTA
constexpr int kRowBytes = 128;      // reduction bytes per stage
constexpr int kThreads = 256;       // warps: 0 TMA, 1 MMA, 2 tail rows, 3 idle, 4-7 epilogue
constexpr int kFirstEpiWarp = 4;
constexpr int kEpilogueWarps = 4;
constexpr uint64_t kDrainTimeoutNs = 200000000ull;

// Wait-site ids reported in the device status word.
enum { kSiteEmpty = 0x21, kSiteFull = 0x22, kSiteTmemEmpty = 0x23, kSiteTmemFull = 0x24, kSiteTail = 0x25 };

struct Params {
    const int32_t* offsets;
    int E, M;
    int out_rows;        // weight gradient: rows of one group's D (K); otherwise unused
    int N;               // columns of D
    int num_kb;          // rows product: stages of the reduction
    int num_n_tiles;
    uint32_t idesc;
    uint8_t* D;          // element size from d_type
    int64_t ldd, d_group;  // row and group stride of D, in elements (d_group: weight gradient)
    int d_type;
    int vec;             // bytes of a store to D (32, 16, or 0: element by element)
    uint8_t* D_scales;
    int nblkN;
    const float* a_scales;
    const float* b_scales;
    const float* bias;
    int* status;
    uint64_t timeout_ns;
};

// kInt8: int8 operands, otherwise 16-bit floats.  kAMn / kBMn: the operand's strided
// axis is the reduction.  kPair: a 2-CTA cluster per tile of 256 rows, otherwise one
// CTA per tile of 128.  BN: columns per tile.  kMx: D in MXFP8.
template <bool kInt8_, bool kAMn_, bool kBMn_, bool kPair_, int BN_, int kStages_, bool kMx_>
struct Config {
    static constexpr bool kInt8 = kInt8_, kAMn = kAMn_, kBMn = kBMn_, kPair = kPair_, kMx = kMx_;
    static constexpr bool kWgrad = kAMn;  // the only product with a ragged reduction
    static constexpr int BN = BN_, kStages = kStages_;
    static constexpr int kCtas = kPair ? 2 : 1;
    static constexpr int TM = BM * kCtas;             // tile rows
    static constexpr int BK = kInt8 ? 128 : 64;       // reduction elements per stage
    static constexpr int kCols = BN / kCtas;          // B columns each CTA loads
    static constexpr int kMnBox = kInt8 ? 128 : 64;   // elements across an MN-major box
    static constexpr int A_BYTES = BM * kRowBytes;
    static constexpr int B_BYTES = kCols * kRowBytes;
    static constexpr int kBoxBytes = kRowBytes * BK;  // an MN-major box: BK rows of 128 bytes
    static constexpr int kFullArrivals = kWgrad && kPair ? 2 : 1;
    static constexpr uint32_t kTmemCols = 2 * BN;
    static constexpr int OFF_A = 0;
    static constexpr int OFF_B = kStages * A_BYTES;
    static constexpr int OFF_BAR = OFF_B + kStages * B_BYTES;
    // barriers: full[S], empty[S], tail[S], tfull[2], tempty[2], drain
    static constexpr int kNumBars = 3 * kStages + 5;
    static constexpr int OFF_MISC = OFF_BAR + kNumBars * 8;
    static constexpr int OFF_TABLE = (OFF_MISC + 64 + 15) / 16 * 16;
    // The table takes 3 words per group behind OFF_TABLE; the launch sizes it.
    static constexpr int smem_bytes(int E) { return OFF_TABLE + 4 * (3 * E + 1) + 1024; }
    static_assert(OFF_TABLE + 4 * (3 * kMaxGroups + 1) + 1024 <= 232448, "shared memory of one block");
    static_assert(kCols % (kBMn ? kMnBox : 8) == 0, "whole boxes of B");
};

// Row ranges of the groups and the number of tiles before each.
struct Table {
    const int *lo, *hi, *first;  // first[E] is the number of tiles of all groups
};

struct Tile {
    int e;
    int lo, hi;  // the group's rows
    int m0, n0;  // tile origin: row within the group (weight gradient: row of D[e]), column
};

// The tiles of one CTA (pair): t, t + stride, ... in group order, M fastest within
// panels of kPanelM tiles, so that the tiles in flight share A rows and B columns in L2.
template <class C>
struct Walk {
    static constexpr int kPanelM = 8;
    int t, stride, e = 0;
    __device__ __forceinline__ Walk(int first, int step) : t(first), stride(step) {}
    __device__ __forceinline__ bool next(const Params& p, const Table& tab, Tile& x)
    {
        if (t >= tab.first[p.E]) return false;
        while (tab.first[e + 1] <= t) ++e;
        const int r = t - tab.first[e];
        x.e = e;
        x.lo = tab.lo[e];
        x.hi = tab.hi[e];
        const int rows = C::kWgrad ? p.out_rows : x.hi - x.lo;
        const int mt = (rows + C::TM - 1) / C::TM;
        const int per_panel = kPanelM * p.num_n_tiles;
        const int panel = r / per_panel;
        const int q = r - panel * per_panel;
        const int h = min(kPanelM, mt - panel * kPanelM);
        const int nt = q / h;
        x.n0 = nt * C::BN;
        x.m0 = (panel * kPanelM + q - nt * h) * C::TM;
        t += stride;
        return true;
    }
    // Stages of the reduction of a tile.
    __device__ __forceinline__ static int stages(const Params& p, const Tile& x)
    {
        return C::kWgrad ? (x.hi - x.lo + C::BK - 1) / C::BK : p.num_kb;
    }
    // Weight gradient: rows of the last stage that belong to the group, 0 if no row
    // behind them needs zeroing (an MMA takes 16 rows, and MMAs past the end are left out).
    __device__ __forceinline__ static int tail_rows(const Tile& x)
    {
        const int rem = (x.hi - x.lo) % C::BK;
        return C::kWgrad && rem % 16 != 0 ? rem : 0;
    }
};

// Groups' bounds -> the table in shared memory.  Bounds are clamped to [0, M] and to
// non-negative lengths, so that no value of offsets leads outside the operands.
template <class C>
__device__ void build_table(const Params& p, int* lo, int* hi, int* first, int* scratch)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kPer = kMaxGroups / kThreads;
    int count[kPer];
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * kPer + i;
        count[i] = 0;
        if (e < p.E) {
            int a = 0, b = p.M;
            if (p.offsets != nullptr) {
                a = min(max(p.offsets[e], 0), p.M);
                b = min(max(p.offsets[e + 1], a), p.M);
            }
            lo[e] = a;
            hi[e] = b;
            const int rows = C::kWgrad ? p.out_rows : b - a;
            count[i] = (rows + C::TM - 1) / C::TM * p.num_n_tiles;
        }
        sum += count[i];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += scratch[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * kPer + i;
        if (e < p.E) {
            first[e] = before;
            before += count[i];
            if (e == p.E - 1) first[p.E] = before;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16)
{
    uint32_t r;
    if (bf16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void st_global_32b(void* p, const uint32_t* w)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// Store nwords (a multiple of 8) 32-bit words at dst with stores of p.vec bytes.
template <int kWords>
__device__ __forceinline__ void store_words(uint8_t* dst, const uint32_t (&w)[kWords], int vec)
{
    if (vec == 32) {
#pragma unroll
        for (int i = 0; i < kWords; i += 8) st_global_32b(dst + 4 * i, w + i);
    } else {
#pragma unroll
        for (int i = 0; i < kWords; i += 4)
            *reinterpret_cast<uint4*>(dst + 4 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
}

// 32 columns (the first `valid` of them inside N) of one row of D, rounded once from
// FP32 to D's type.
__device__ __forceinline__ void store_row_chunk(const Params& p, int64_t element, int valid, const float (&v)[32])
{
    if (p.d_type == MPK_TYPE_F32) {
        float* dst = reinterpret_cast<float*>(p.D) + element;
        if (valid == 32 && p.vec) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
            store_words(reinterpret_cast<uint8_t*>(dst), w, p.vec);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i < valid) dst[i] = v[i];
        }
    } else {
        const bool bf16 = p.d_type == MPK_TYPE_BF16;
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.D) + element;
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = pack16(v[2 * i], v[2 * i + 1], bf16);
        if (valid == 32 && p.vec) {
            store_words(reinterpret_cast<uint8_t*>(dst), w, p.vec);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i < valid) dst[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

// One MX block of a row: the framework's block rule (mx_block_scale), as in the MXFP8
// GEMM's epilogue.  Columns past N are zeros (their B columns were filled with zeros).
__device__ __forceinline__ void store_mx_chunk(const Params& p, int64_t row, int col0, int valid, const float (&v)[32])
{
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(v[i]));  // NaN ignored
    float inv;
    const uint32_t s = mx_block_scale(amax, inv);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint2 q = quantize8(v + 8 * i, inv);
        w[2 * i] = q.x;
        w[2 * i + 1] = q.y;
    }
    uint8_t* dst = p.D + row * p.ldd + col0;
    if (valid == 32 && p.vec) {
        store_words(dst, w, p.vec);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < valid) dst[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
    }
    p.D_scales[row * p.nblkN + col0 / 32] = (uint8_t)s;
}

template <class C>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    if constexpr (C::kInt8) {
        if constexpr (C::kPair) umma_i8_pair(d, a, b, idesc, acc);
        else umma_i8(d, a, b, idesc, acc);
    } else {
        if constexpr (C::kPair) umma_bf16_pair(d, a, b, idesc, acc);
        else umma_bf16(d, a, b, idesc, acc);
    }
}

template <class C>
__device__ __forceinline__ void commit_all(uint32_t bar)
{
    if constexpr (C::kPair) umma_commit_pair_mc(bar, 0x3);
    else umma_commit(bar);
}

template <class C>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Params p)
{
    constexpr int S = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar0 = sbase + C::OFF_BAR;
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (S + s); };
    auto tail = [&](int s) { return bar0 + 8u * (2 * S + s); };
    auto tfull = [&](int a) { return bar0 + 8u * (3 * S + a); };
    auto tempty = [&](int a) { return bar0 + 8u * (3 * S + 2 + a); };
    const uint32_t drain = bar0 + 8u * (3 * S + 4);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
    volatile int* never_abort = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 8);
    int* scratch = reinterpret_cast<int*>(smem + C::OFF_MISC + 16);
    int* t_lo = reinterpret_cast<int*>(smem + C::OFF_TABLE);
    int* t_hi = t_lo + p.E;
    int* t_first = t_hi + p.E;
    const Table tab{t_lo, t_hi, t_first};

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = C::kPair ? cluster_ctarank() : 0u;
    const int unit = C::kPair ? (int)cluster_id_x() : (int)blockIdx.x;
    const int nunits = C::kPair ? (int)nclusters_x() : (int)gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full(s), C::kFullArrivals);
            mbar_init(empty(s), 1);
            mbar_init(tail(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull(a), 1);
            mbar_init(tempty(a), C::kCtas * kEpilogueWarps);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        *never_abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (C::kPair) {
            tmem_alloc_pair(smem_u32(tmem_holder), C::kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_holder), C::kTmemCols);
            tmem_relinquish();
        }
    }
    // A kernel of this library may still be running in front of this one (codes,
    // scales or a padded operand): nothing global is touched before it has completed.
    wait_for_prerequisite_grid();
    build_table<C>(p, t_lo, t_hi, t_first, scratch);
    tc_fence_before();
    if constexpr (C::kPair) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    bool producer_aborted = false;
    Walk<C> walk(unit, nunits);
    Tile x;

    if (warp == 0) {
        // ------------------------------ TMA producer -------------------------------
        if (lane == 0) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            uint32_t last_tail = 0, tail_ph = 0;  // per stage: its last use went through tail(s); uses so, mod 2
            bool ok = true;
            while (ok && walk.next(p, tab, x)) {
                const int nkb = walk.stages(p, x);
                const int tail_rows = walk.tail_rows(x);
                const int m = x.m0 + BM * (int)rank;
                const int n = x.n0 + C::kCols * (int)rank;
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!mbar_wait(empty(s), ph ^ 1u, abort_flag, p.status, kSiteEmpty, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    uint32_t bar;
                    last_tail &= ~(1u << s);
                    if (C::kWgrad && tail_rows > 0 && kb == nkb - 1) {
                        // This CTA's tail warp takes the stage first.
                        bar = tail(s);
                        last_tail |= 1u << s;
                        tail_ph ^= 1u << s;
                        mbar_arrive_expect_tx(bar, C::A_BYTES + C::B_BYTES);
                        if constexpr (C::kPair) bar = mapa_shared(bar, rank);
                    } else {
                        if (rank == 0) {
                            mbar_arrive_expect_tx(full(s), C::kCtas * (C::A_BYTES + C::B_BYTES));
                            if (C::kFullArrivals == 2) mbar_arrive(full(s));
                        }
                        bar = full(s);
                        if constexpr (C::kPair) bar = mapa_shared(bar, 0);
                    }
                    const uint32_t a = sbase + C::OFF_A + s * C::A_BYTES;
                    const uint32_t b = sbase + C::OFF_B + s * C::B_BYTES;
                    auto load_a = [&](uint32_t dst, int c0, int c1) {
                        if constexpr (C::kPair) tma_load_2d_pair(dst, &tmap_a, bar, c0, c1);
                        else tma_load_2d(dst, &tmap_a, bar, c0, c1);
                    };
                    auto load_b = [&](uint32_t dst, int c0, int c1, int c2) {
                        if constexpr (C::kPair) tma_load_3d_pair(dst, &tmap_b, bar, c0, c1, c2);
                        else tma_load_3d(dst, &tmap_b, bar, c0, c1, c2);
                    };
                    const int k0 = kb * C::BK;
                    if constexpr (C::kAMn) {
#pragma unroll
                        for (int j = 0; j < BM / C::kMnBox; ++j)
                            load_a(a + j * C::kBoxBytes, m + j * C::kMnBox, x.lo + k0);
                    } else {
                        load_a(a, k0, x.lo + m);
                    }
                    if constexpr (C::kBMn) {
#pragma unroll
                        for (int j = 0; j < C::kCols / C::kMnBox; ++j)
                            load_b(b + j * C::kBoxBytes, n + j * C::kMnBox, C::kWgrad ? x.lo + k0 : k0,
                                   C::kWgrad ? 0 : x.e);
                    } else {
                        load_b(b, k0, n, x.e);
                    }
                    ++issued;
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok) {
                // Copies in flight land before shared memory is released.
                producer_aborted = true;
                const int outstanding = issued < S ? issued : S;
                int ss = s;
                uint32_t pp = ph;
                for (int i = 0; i < outstanding; ++i) {
                    if (--ss < 0) { ss = S - 1; pp ^= 1u; }
                    if ((last_tail >> ss) & 1u)
                        mbar_wait(tail(ss), ((tail_ph >> ss) & 1u) ^ 1u, never_abort, nullptr, 0, kDrainTimeoutNs);
                    else if (rank == 0)
                        mbar_wait(full(ss), pp, never_abort, nullptr, 0, kDrainTimeoutNs);
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------- MMA issuer --------------------------------
        if (rank == 0 && lane == 0) {
            int s = 0, it = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (; ok && walk.next(p, tab, x); ++it) {
                const int nkb = walk.stages(p, x);
                const int acc = it & 1;
                if (!mbar_wait(tempty(acc), ((uint32_t)(it >> 1) & 1u) ^ 1u, abort_flag, p.status, kSiteTmemEmpty,
                               p.timeout_ns)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(acc * C::BN);
                const int rem = (x.hi - x.lo) % C::BK;
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!mbar_wait(full(s), ph, abort_flag, p.status, kSiteFull, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    int steps = 4;
                    if (C::kWgrad && kb == nkb - 1 && rem != 0) {
                        steps = (rem + 15) / 16;
                        fence_acq_rel_cluster();  // the tail warps' zeros, of both CTAs
                    }
                    tc_fence_after();
                    const uint32_t a = sbase + C::OFF_A + s * C::A_BYTES;
                    const uint32_t b = sbase + C::OFF_B + s * C::B_BYTES;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (C::kWgrad && k >= steps) break;
                        // A step is 32 bytes along a K-major row, or BK / 4 rows of an MN-major box.
                        constexpr uint32_t kMnStep = C::BK / 4 * kRowBytes;
                        const uint64_t ad = C::kAMn ? umma_smem_desc_sw128(a + k * kMnStep, C::kBoxBytes, 1024)
                                                    : umma_smem_desc_sw128(a + k * 32, 16, 1024);
                        const uint64_t bd = C::kBMn ? umma_smem_desc_sw128(b + k * kMnStep, C::kBoxBytes, 1024)
                                                    : umma_smem_desc_sw128(b + k * 32, 16, 1024);
                        mma<C>(d, ad, bd, p.idesc, (kb != 0 || k != 0) ? 1u : 0u);
                    }
                    commit_all<C>(empty(s));
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                if (!ok) break;
                commit_all<C>(tfull(acc));
            }
            if constexpr (C::kPair) umma_commit_pair(drain);
            else umma_commit(drain);
            mbar_wait(drain, 0, never_abort, nullptr, 0, kDrainTimeoutNs);
        }
    } else if (C::kWgrad && warp == 2) {
        // ------- tail rows: zeros behind the group's end, in A and in B -------
        // A zero in A alone would leave NaN where the next group's B holds NaN.
        int s = 0;
        uint32_t phases = 0;  // parity of each stage's tail barrier
        const uint32_t full0 = C::kPair ? mapa_shared(full(0), 0) : full(0);
        bool ok = true;
        while (ok && walk.next(p, tab, x)) {
            const int nkb = walk.stages(p, x);
            const int rows = walk.tail_rows(x);
            if (nkb == 0) continue;
            const int last = (s + nkb - 1) % S;
            s = (last + 1) % S;
            if (rows == 0) continue;
            ok = mbar_wait(tail(last), (phases >> last) & 1u, abort_flag, p.status, kSiteTail, p.timeout_ns);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            phases ^= 1u << last;
            const int end = (rows + 15) / 16 * 16;
            // 128-byte rows of each box: the swizzle permutes within a row, so whole rows are plain.
            constexpr int kABoxes = BM / C::kMnBox, kBBoxes = C::kCols / C::kMnBox;
            const int chunks = (end - rows) * 8;
            for (int j = 0; j < kABoxes + kBBoxes; ++j) {
                uint8_t* box = j < kABoxes ? smem + C::OFF_A + last * C::A_BYTES + j * C::kBoxBytes
                                           : smem + C::OFF_B + last * C::B_BYTES + (j - kABoxes) * C::kBoxBytes;
                for (int i = lane; i < chunks; i += 32)
                    reinterpret_cast<uint4*>(box + rows * kRowBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if constexpr (C::kPair) mbar_arrive_cluster_release(full0 + 8u * last);
                else mbar_arrive(full0 + 8u * last);
            }
        }
    } else if (warp >= kFirstEpiWarp) {
        // -------------------------------- epilogue ---------------------------------
        const int quad = warp & 3;
        const int r = quad * 32 + lane;  // accumulator row
        const uint32_t tempty0 = C::kPair ? mapa_shared(tempty(0), 0) : tempty(0);
        for (int it = 0; walk.next(p, tab, x); ++it) {
            const int acc = it & 1;
            const int rows = C::kWgrad ? p.out_rows : x.hi - x.lo;
            const int row = x.m0 + BM * (int)rank + r;  // within the group
            const bool row_ok = row < rows;
            const bool warp_ok = x.m0 + BM * (int)rank + quad * 32 < rows;
            const int64_t grow = C::kWgrad ? (int64_t)row : (int64_t)x.lo + row;
            const int64_t base = (C::kWgrad ? x.e * p.d_group : 0) + grow * p.ldd;
            const bool any = walk.stages(p, x) > 0;  // otherwise nothing was accumulated: zeros
            float sa = 0.0f;
            if (C::kInt8 && row_ok) sa = p.a_scales[grow];  // may be written by the kernel in front: no read-only load
            if (!mbar_wait(tfull(acc), (uint32_t)(it >> 1) & 1u, abort_flag, p.status, kSiteTmemFull, p.timeout_ns))
                break;
            tc_fence_after();
            const uint32_t trow = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * C::BN);
            if (warp_ok) {
#pragma unroll 1
                for (int c = 0; c < C::BN / 32; ++c) {
                    const int col0 = x.n0 + 32 * c;
                    if (col0 >= p.N) break;
                    const int valid = min(32, p.N - col0);
                    uint32_t raw[32];
                    if (any) {
                        tmem_ld_32x32b_x32(trow + 32u * c, raw);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) raw[i] = 0u;
                    }
                    float v[32];
                    if constexpr (C::kInt8) {
                        const float* sb = p.b_scales + (int64_t)x.e * p.N + col0;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float b = i < valid ? __ldg(sb + i) : 0.0f;
                            v[i] = __fmul_rn(__fmul_rn((float)(int)raw[i], sa), b);
                            if (p.bias != nullptr && i < valid) v[i] = __fadd_rn(v[i], __ldg(p.bias + col0 + i));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]);
                    }
                    if (row_ok) {
                        if constexpr (C::kMx) store_mx_chunk(p, grow, col0, valid, v);
                        else store_row_chunk(p, base + col0, valid, v);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (C::kPair) mbar_arrive_cluster(tempty0 + 8u * acc);
                else mbar_arrive(tempty0 + 8u * acc);
            }
        }
    }

    if (producer_aborted) {
        // A copy of the other CTA may still be landing after rank 0 stopped expecting it.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 100000ull) {
        }
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (C::kPair) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (C::kPair) tmem_dealloc_pair(tmem_base, C::kTmemCols);
        else tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

}  // namespace product

// ----------------------------------------------------------------------------
// Host side
// ----------------------------------------------------------------------------
namespace {

std::mutex g_attr_mu;

template <class C>
int launch_config(const ProductArgs& a, product::Params& p, int64_t max_tiles, cudaStream_t stream, int dev)
{
    using namespace product;
    static bool attr_set[64] = {};
    const int eb = C::kInt8 ? 1 : 2;
    CUtensorMap ta{}, tb{};
    const CUtensorMapDataType dt = C::kInt8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : a.ab_type == MPK_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int reduction = C::kWgrad ? a.M : a.K;
    if (reduction > 0) {  // otherwise no load is issued
        const uint64_t adims[2] = {(uint64_t)a.K, (uint64_t)a.M};
        const uint64_t astr[1] = {(uint64_t)a.lda * eb};
        const uint32_t abox[2] = {(uint32_t)(C::kAMn ? C::kMnBox : C::BK), (uint32_t)(C::kAMn ? C::BK : BM)};
        if (int rc = encode_tensor_map(&ta, dt, a.A, 2, adims, astr, abox)) return rc;
        const int b_inner = C::kBMn ? a.N : a.K;
        const int b_rows = C::kWgrad ? a.M : (C::kBMn ? a.K : a.N);
        const uint64_t bdims[3] = {(uint64_t)b_inner, (uint64_t)b_rows, (uint64_t)(C::kWgrad ? 1 : a.E)};
        const uint64_t bstr[2] = {(uint64_t)a.ldb * eb, (uint64_t)a.ldb * eb * (uint64_t)b_rows};
        const uint32_t bbox[3] = {(uint32_t)(C::kBMn ? C::kMnBox : C::BK), (uint32_t)(C::kBMn ? C::BK : C::kCols), 1u};
        if (int rc = encode_tensor_map(&tb, dt, a.B, 3, bdims, bstr, bbox)) return rc;
    }
    p.num_kb = (a.K + C::BK - 1) / C::BK;
    p.num_n_tiles = (a.N + C::BN - 1) / C::BN;
    if (C::kInt8)
        p.idesc = (2u << 4) | (1u << 7) | (1u << 10);  // S32 sums, signed 8-bit A and B
    else
        p.idesc = (1u << 4) | (a.ab_type == MPK_TYPE_BF16 ? (1u << 7) | (1u << 10) : 0u);  // FP32 sums
    p.idesc |= ((C::kAMn ? 1u : 0u) << 15) | ((C::kBMn ? 1u : 0u) << 16) | ((uint32_t)(C::BN >> 3) << 17) |
               ((uint32_t)(C::TM >> 4) << 24);

    // The walk counts tiles in 32 bits.
    const int64_t m_tiles = C::kWgrad ? (int64_t)a.E * ((a.K + C::TM - 1) / C::TM)
                                      : (int64_t)a.M / C::TM + std::min(a.E, a.M);
    const int64_t tiles = m_tiles * p.num_n_tiles;
    if (tiles > INT32_MAX / 2) {
        set_last_error("product of more than 2^30 tiles (M=%d N=%d K=%d, %d groups)", a.M, a.N, a.K, a.E);
        return MPK_ERR_UNSUPPORTED;
    }
    const int smem = C::smem_bytes(a.E);
    const auto kernel = product_kernel<C>;
    {
        std::lock_guard<std::mutex> lk(g_attr_mu);
        if (!attr_set[dev]) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       C::smem_bytes(kMaxGroups));
            if (e != cudaSuccess) {
                set_last_error("cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
                return (int)e;
            }
            attr_set[dev] = true;
        }
    }
    const int64_t units = std::min<int64_t>(tiles, device_sm_count() / C::kCtas);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)units * C::kCtas, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (C::kPair) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (a.after_kernel) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ta, tb, p);
    if (e == cudaErrorInvalidValue || e == cudaErrorLaunchOutOfResources) {
        // A context re-created by cudaDeviceReset has lost the shared-memory attribute.
        cudaGetLastError();
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem_bytes(kMaxGroups)) ==
            cudaSuccess)
            e = cudaLaunchKernelEx(&cfg, kernel, ta, tb, p);
    }
    if (e != cudaSuccess) {
        set_last_error("product launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MPK_SUCCESS;
}

}  // namespace

bool product_tma_ok(const void* p, int64_t ld, int elem_bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * elem_bytes % 16 == 0;
}

int launch_product(const ProductArgs& a, cudaStream_t stream)
{
    using namespace product;
    int dev = 0;
    int* status = nullptr;
    if (int rc = kernel_device_context(dev, &status)) return rc;
    Params p = {};
    p.offsets = a.offsets;
    p.E = a.E;
    p.M = a.M;
    p.out_rows = a.K;
    p.N = a.N;
    p.D = static_cast<uint8_t*>(a.D);
    p.ldd = a.ldd;
    p.d_group = (int64_t)a.K * a.ldd;
    p.d_type = a.d_type;
    p.D_scales = a.D_scales;
    p.nblkN = (a.N + 31) / 32;
    p.a_scales = a.a_scales;
    p.b_scales = a.b_scales;
    p.bias = a.bias;
    p.status = status;
    p.timeout_ns = wait_timeout_ns();
    const int db = a.d_type == kTypeMxfp8 ? 1 : a.d_type == MPK_TYPE_F32 ? 4 : 2;
    p.vec = 0;
    for (int v : {16, 32})
        if (reinterpret_cast<uintptr_t>(a.D) % v == 0 && a.ldd * db % v == 0) p.vec = v;
    if (a.wgrad)
        return launch_config<Config<false, true, true, true, 256, 6, false>>(a, p, 0, stream, dev);
    // Tiles of 256 rows when groups have that many on average.
    const bool pair = (int64_t)a.M >= 192 * (int64_t)a.E;
    if (a.ab_type == kTypeInt8) {
        if (a.b_nk) {
            if (pair) return launch_config<Config<true, false, false, true, 256, 6, false>>(a, p, 0, stream, dev);
            return launch_config<Config<true, false, false, false, 128, 6, false>>(a, p, 0, stream, dev);
        }
        if (pair) return launch_config<Config<true, false, true, true, 256, 6, false>>(a, p, 0, stream, dev);
        return launch_config<Config<true, false, true, false, 128, 6, false>>(a, p, 0, stream, dev);
    }
    if (a.d_type == kTypeMxfp8) {
        if (pair) return launch_config<Config<false, false, true, true, 256, 6, true>>(a, p, 0, stream, dev);
        return launch_config<Config<false, false, true, false, 128, 6, true>>(a, p, 0, stream, dev);
    }
    if (a.b_nk) {
        if (pair) return launch_config<Config<false, false, false, true, 256, 6, false>>(a, p, 0, stream, dev);
        return launch_config<Config<false, false, false, false, 128, 6, false>>(a, p, 0, stream, dev);
    }
    if (pair) return launch_config<Config<false, false, true, true, 256, 6, false>>(a, p, 0, stream, dev);
    return launch_config<Config<false, false, true, false, 128, 6, false>>(a, p, 0, stream, dev);
}

}  // namespace mpk
