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
// Orientation.  The columns of D lie on the MMA's M axis (128 per CTA, one tensor-memory
// lane each) and the rows of D on its N axis (one tensor-memory column each).  N can be
// any multiple of 16 up to 256 per MMA, so a group of r rows costs a tile about r wide
// instead of a multiple of 128 or 256: a group of up to 256 rows reads its weights once,
// and a few tokens cost hardly more than the weights' bytes.  A warp then holds 32
// neighbouring columns of one row of D and stores them together, whatever D's alignment.
//
// The groups' bounds are read from device memory, so that a router's result needs no
// copy to the host: every CTA scans them into shared memory (row ranges and a running
// count of tiles) and the clusters walk the tiles of all groups with a stride of the grid.
//
// Operands stream by TMA into a ring of 128-byte-wide stages (64 16-bit or 128 8-bit
// elements of the reduction), swizzled as the MMA reads them, in whatever order they
// are stored: the reduction axis may be the contiguous one (K-major) or the strided
// one (MN-major).  A group's rows start anywhere: a load may begin at any row, and rows
// of the next group that land in a tile only make accumulator columns that are not
// stored.  Where the ragged axis is the reduction (weight gradient) the rows behind the
// group's end are zeroed in shared memory before the last MMAs.
//
// Accumulators live in tensor memory, two of them, so that a tile's epilogue runs
// under the next tile's MMAs.  FP32 sums for the 16-bit types, 32-bit integer sums
// (exact: the host refuses a K at which they could overflow) for int8.  Where there are
// fewer tiles than SMs, the CTAs of a cluster share a tile's reduction and join their
// sums through distributed shared memory in a fixed order (splits).
//
// What bounds it (B200): few rows, the weights' bytes (16 tokens through 16 experts of
// 2048x2048 BF16 in 24 us: 5.6 TB/s over the whole call, of the 6.5 a copy reaches, its launch
// and first loads included); many rows, the tensor pipe and, over seconds, the
// power cap (int8 4096x12288x4096 in 128 us, 3.2 POP/s, the pipe busy 82 % of the time; BF16
// with one group 262 to 269 us, 1.53 to 1.57 PFLOP/s); a short reduction, the epilogue's
// stores (weight gradient of 32 x 2048x2816 BF16 in 87 us, 4.2 TB/s).
//
// Every mbarrier wait is bounded (mpk::mbar_wait); on expiry the CTA raises an abort
// flag (where a cluster joins its sums, that of all its CTAs), records a status code, drains
// what it has in flight and leaves.  What it has not stored by then stays as it was.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "int8_codes.cuh"
#include "mpk.h"
#include "mpk_internal.h"
#include "mpk_ptx.cuh"

namespace mpk {
namespace product {

constexpr int kCols = 128;          // columns of D per CTA: tensor-memory lanes
constexpr int kMaxRows = 256;       // rows of D per tile: tensor-memory columns of an accumulator
constexpr int kRowBytes = 128;      // reduction bytes per stage
constexpr int kTurnStride = 36;     // floats between the rows of a turned 32 x 32 chunk
constexpr int kMaxStages = 12;
constexpr int kFirstEpiWarp = 4;    // warps: 0 TMA, 1 MMA, 2 tail rows, 3 idle, then the epilogue's
constexpr int kMaxWarps = 20;
constexpr int kFuseWarps = 8;       // epilogue warps of a product that quantizes its rows
constexpr int P_BYTES = kCols * kRowBytes;  // columns operand per CTA and stage
constexpr uint64_t kDrainTimeoutNs = 200000000ull;

// Shared memory behind the ring: barriers full, empty, tail [kMaxStages], tfull[2],
// tempty[2], drain, codes; flags and scan scratch; row scales; the table of groups (3
// words each).
constexpr int kNumBars = 3 * kMaxStages + 6;
constexpr int kMiscOffset = kNumBars * 8;
constexpr int kScaleOffset = (kMiscOffset + 16 + 4 * 2 * kMaxWarps + 15) / 16 * 16;  // 32 row scales per warp
constexpr int kCodesOffset = kScaleOffset + 32 * 4 * (kMaxWarps - kFirstEpiWarp);  // fused quantizer: amax and scale per row
constexpr int kFusedRows = 16;      // most rows of a product that quantizes them itself
constexpr int kTableOffset = kCodesOffset + 2 * 4 * kFusedRows;

constexpr int control_bytes(int E) { return kTableOffset + 4 * (3 * E + 1); }

// Wait-site ids reported in the device status word.
enum { kSiteEmpty = 0x21, kSiteFull = 0x22, kSiteTmemEmpty = 0x23, kSiteTmemFull = 0x24, kSiteTail = 0x25,
       kSiteCodes = 0x26 };

struct Params {
    const int32_t* offsets;
    int E, M;
    int out_rows;        // weight gradient: rows of one group's D (K); otherwise unused
    int N;               // columns of D
    int num_kb;          // rows product: stages of the reduction
    int num_n_tiles;
    int have_operands;   // the reduction is not empty: the operands' tensor maps are set
    int splits;          // CTAs (pairs) of a cluster that share a tile's reduction
    int read_once;       // most of P is read by one tile only
    int early;           // the kernel in front writes nothing but Q and its scales
    int ring_bytes;      // the ring; stage_bytes of the widest tile cuts it into stages
    int parts_in_ring, parts_offset;  // splits: where their sums meet (offset from the barriers)
    // Fused quantizer: x [M][K], and the bytes its codes take behind the ring.
    const void* x;
    int64_t ldx;
    int x_type, x_vec;   // x_vec: rows can be read in 16-byte pieces
    int K, codes_bytes;
    int tmem_cols, acc_cols;  // tensor memory allocated, and columns from one accumulator to the next
    uint32_t idesc;      // without N
    uint8_t* D;          // element size from d_type
    int64_t ldd, d_group;  // row and group stride of D, in elements (d_group: weight gradient)
    int d_type;
    int d_vec;           // MXFP8: rows of D are 16-byte aligned; 16-bit D: 4-byte aligned
    uint8_t* D_scales;
    int nblkN;
    const float* a_scales;
    const float* b_scales;
    const float* bias;
    int* status;
    uint64_t timeout_ns;
};

// P is the operand of D's columns (weights; dD in a weight gradient), Q that of D's rows
// (A).  kInt8: int8 operands, otherwise 16-bit floats.  kPMn: P's strided axis is the
// reduction.  kWgrad: weight gradient, both operands MN-major.  kPair: a 2-CTA pair per
// tile of 256 columns, otherwise one CTA per tile of 128.  kMx: D in MXFP8.  kFuse: int8
// codes and scales of up to kFusedRows rows are made from p.x by every CTA itself.
template <bool kInt8_, bool kPMn_, bool kWgrad_, bool kPair_, bool kMx_, bool kFuse_ = false>
struct Config {
    static constexpr bool kFuse = kFuse_;
    static_assert(!kFuse || (kInt8_ && !kPair_), "the fused quantizer is for few rows of int8");
    static constexpr bool kInt8 = kInt8_, kPMn = kPMn_, kWgrad = kWgrad_, kPair = kPair_, kMx = kMx_;
    static_assert(!kWgrad || (kPMn && !kInt8), "a weight gradient's operands are MN-major 16-bit floats");
    static constexpr int kCtas = kPair ? 2 : 1;
    static constexpr int BK = kInt8 ? 128 : 64;       // reduction elements per stage
    static constexpr int kMnBox = kInt8 ? 128 : 64;   // elements across an MN-major box
    static constexpr int kBoxBytes = kRowBytes * BK;  // an MN-major box: BK rows of 128 bytes
    static constexpr int kRowStep = 16 * kCtas;       // a tile's rows are a multiple
    // A weight gradient often has more to store than to multiply: twice the epilogue (32 x
    // 2048x2816 BF16 of 4096 rows: 123 -> 87 us), which costs products with a long reduction
    // 2 to 3 %.
    static constexpr int kEpiWarps = kWgrad ? 16 : 8;
    static constexpr int kTurns = kEpiWarps / 4;      // warps that take turns at chunks of 32 rows
    static constexpr int kThreads = 32 * (kFirstEpiWarp + kEpiWarps);
    static constexpr int kFullArrivals = kWgrad && kPair ? 2 : 1;
};

// Row ranges of the groups and the number of tiles before each.
struct Table {
    const int *lo, *hi, *first;  // first[E] is the number of tiles of all groups
};

// Rows of a tile of a group of `rows`: its share of equal tiles of at most kMaxRows,
// rounded up to what the MMA takes.
template <class C>
__host__ __device__ __forceinline__ int tile_width(int rows)
{
    if (rows > kMaxRows) {
        const int mt = (rows + kMaxRows - 1) / kMaxRows;
        rows = (rows + mt - 1) / mt;
    }
    return (rows + C::kRowStep - 1) / C::kRowStep * C::kRowStep;
}

// Stage of a product whose widest tile has `width` rows.  The groups' real sizes decide
// it, not the host's bound: with few rows per group a stage is little more than its
// weights, and the ring keeps more of them in flight.
template <class C>
__host__ __device__ __forceinline__ int stage_bytes(int width)
{
    return P_BYTES + (C::kFuse ? 0 : width / C::kCtas * kRowBytes);
}

struct Tile {
    int e;
    int lo, hi;     // the group's rows
    int r0, rows;   // rows of D: first one within the group (weight gradient: within D[e]) and count
    int width;      // rows rounded up to what the MMA takes
    int n0;         // first column
};

// ceil(2^32 / h) for the row tiles h of a panel.
__constant__ const uint32_t kReciprocal[17] = {
    0u,          0u,          0x80000000u, 0x55555556u, 0x40000000u, 0x33333334u, 0x2AAAAAABu, 0x24924925u, 0x20000000u,
    0x1C71C71Du, 0x1999999Au, 0x1745D175u, 0x15555556u, 0x13B13B14u, 0x12492493u, 0x11111112u, 0x10000000u};

// The tiles of one cluster: t, t + stride, ... in group order, row tiles fastest within
// panels of kPanel, so that the tiles in flight share rows and columns in L2.  A group's
// rows are cut into equal tiles of at most kMaxRows.
template <class C>
struct Walk {
    static constexpr int kPanel = 16;
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
        const int mt = (rows + kMaxRows - 1) / kMaxRows;
        const int per = C::kWgrad ? kMaxRows : tile_width<C>(rows);
        // The epilogue of a short reduction waits for this: no division where there is one
        // panel (the usual case), and one by h as a multiplication, exact below 2^28.
        int panel = 0, q = r, h = mt;
        if (mt > kPanel) {
            const int per_panel = kPanel * p.num_n_tiles;
            panel = r / per_panel;
            q = r - panel * per_panel;
            h = min(kPanel, mt - panel * kPanel);
        }
        const int nt = h == 1 ? q : (int)__umulhi((uint32_t)q, kReciprocal[h]);
        x.n0 = nt * kCols * C::kCtas;
        x.r0 = (panel * kPanel + q - nt * h) * per;
        x.rows = min(per, rows - x.r0);
        x.width = per;
        t += stride;
        return true;
    }
    // Stages [k0, k1) of a tile's reduction that split s of p.splits takes.
    __device__ __forceinline__ static void stages(const Params& p, const Tile& x, int s, int& k0, int& k1)
    {
        const int n = all_stages(p, x);
        k0 = p.splits == 1 ? 0 : (int)((int64_t)n * s / p.splits);
        k1 = p.splits == 1 ? n : (int)((int64_t)n * (s + 1) / p.splits);
    }
    __device__ __forceinline__ static int all_stages(const Params& p, const Tile& x)
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

// Groups' bounds -> the table in shared memory, and the widest tile's rows (both to be read
// after a __syncthreads).  Bounds are clamped to [0, M] and to
// non-negative lengths, so that no value of offsets leads outside the operands.
template <class C>
__device__ void build_table(const Params& p, int* lo, int* hi, int* first, int* scratch, int* widest)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.E == 1) {
        if (tid == 0) {
            int a = 0, b = p.M;
            if (p.offsets != nullptr) {
                a = min(max(p.offsets[0], 0), p.M);
                b = min(max(p.offsets[1], a), p.M);
            }
            lo[0] = a;
            hi[0] = b;
            first[0] = 0;
            first[1] = ((C::kWgrad ? p.out_rows : b - a) + kMaxRows - 1) / kMaxRows * p.num_n_tiles;
            *widest = b > a ? tile_width<C>(b - a) : C::kRowStep;
        }
        return;
    }
    constexpr int kThreads = C::kThreads, kPer = (kMaxGroups + kThreads - 1) / kThreads;
    int count[kPer];
    int sum = 0, wide = C::kRowStep;
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
            count[i] = (rows + kMaxRows - 1) / kMaxRows * p.num_n_tiles;
            if (rows > 0) wide = max(wide, tile_width<C>(rows));
        }
        sum += count[i];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += v;
    }
    wide = (int)__reduce_max_sync(0xFFFFFFFFu, (unsigned)wide);
    if (lane == 31) {
        scratch[warp] = incl;
        scratch[kThreads / 32 + warp] = wide;
    }
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += scratch[w];
    if (tid == 0) {
        for (int w = 0; w < kThreads / 32; ++w) wide = max(wide, scratch[kThreads / 32 + w]);
        *widest = wide;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = tid * kPer + i;
        if (e < p.E) {
            first[e] = before;
            before += count[i];
            if (e == p.E - 1) first[p.E] = before;
        }
    }
}

// The fused quantizer: the epilogue warps (ew of kFuseWarps) make the codes of rows
// 0 .. M - 1 for the reduction's elements [kfirst, klast) in shared memory, as TMA would
// have laid them out (a block of kFusedRows rows per stage, 128-byte swizzle), and the
// rows' scales.  Every CTA reads whole rows of x for their largest magnitude, while its
// first stages of weights are on their way.
template <class T>
__device__ __forceinline__ void make_codes(const Params& p, int ew, int lane, int kfirst, int klast, uint8_t* codes,
                                           uint32_t* amax_bits, float* scales)
{
    constexpr int V = T::kVec;
    const int M = p.M;
    const int warps = M == 1 ? 8 : M == 2 ? 4 : M <= 4 ? 2 : 1;  // of one row
    const int nvec = p.x_vec ? p.K / V : 0;
    const int start = (ew % warps) * 32 + lane, stride = warps * 32;
    if (ew == 0 && lane < kFusedRows) amax_bits[lane] = 0u;
    __syncwarp();
    named_bar_sync(1, 32 * kFuseWarps);
    for (int m = ew / warps; m < M; m += kFuseWarps / warps) {
        const typename T::T* row = static_cast<const typename T::T*>(p.x) + m * p.ldx;
        uint32_t a = 0u;
#pragma unroll 4
        for (int i = start; i < nvec; i += stride) {
            float v[V];
            T::widen(load_16b(reinterpret_cast<const uint4*>(row) + i), v);
#pragma unroll
            for (int j = 0; j < V; ++j) a = max(a, int8::magnitude(v[j]));
        }
        for (int k = nvec * V + start; k < p.K; k += stride) a = max(a, int8::magnitude(T::widen(row[k])));
        a = __reduce_max_sync(0xFFFFFFFFu, a);
        if (lane == 0) atomicMax(&amax_bits[m], a);  // a maximum has no order
    }
    __syncwarp();
    named_bar_sync(1, 32 * kFuseWarps);
    for (int m = ew / warps; m < M; m += kFuseWarps / warps) {
        const typename T::T* row = static_cast<const typename T::T*>(p.x) + m * p.ldx;
        const int8::RowScale rs = int8::row_scale(amax_bits[m]);
        if (start == 0) scales[m] = rs.scale;
        auto at = [&](int k) {  // byte of element k (V elements from a multiple of V stay together)
            const int q = k - kfirst, in = q & 127;
            return codes + (q >> 7) * (kFusedRows * kRowBytes) + m * kRowBytes + ((((in >> 4) ^ m) & 7) << 4) +
                   (in & 15);
        };
        const int vlast = min(klast / V, nvec);
#pragma unroll 2
        for (int i = kfirst / V + start; i < vlast; i += stride) {
            float v[V];
            T::widen(load_16b(reinterpret_cast<const uint4*>(row) + i), v);
            uint32_t* dst = reinterpret_cast<uint32_t*>(at(i * V));
#pragma unroll
            for (int j = 0; j < V; j += 4) dst[j / 4] = int8::pack4(v + j, rs.inv);
        }
        for (int k = max(kfirst, vlast * V) + start; k < klast; k += stride)
            *at(k) = rs.inv == 0.0f ? (uint8_t)0 : (uint8_t)int8::code_bits(T::widen(row[k]), rs.inv);
    }
    fence_proxy_async_smem();
    __syncwarp();
    named_bar_sync(1, 32 * kFuseWarps);
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

// One lane's column of D, and how its sums become elements of D.
template <class C>
struct Column {
    const Params& p;
    int n;          // column
    bool ok;        // inside N
    float sb, bias; // int8: the column's scale and bias

    __device__ __forceinline__ Column(const Params& q, const Tile& x, int col)
        : p(q), n(col), ok(col < q.N), sb(0.0f), bias(-0.0f)
    {
        if (C::kInt8 && ok) {
            sb = p.b_scales[(int64_t)x.e * p.N + n];
            if (p.bias != nullptr) bias = p.bias[n];
        }
    }

    // Adding -0.0f where there is no bias changes no value.
    __device__ __forceinline__ float value(uint32_t raw, float sa) const
    {
        if constexpr (C::kInt8) return __fadd_rn(__fmul_rn(__fmul_rn((float)(int)raw, sa), sb), bias);
        return __uint_as_float(raw);
    }

    // One MX block of row `row` held by the 32 lanes of the warp, which call it together with
    // neighbouring columns, the first a multiple of 32.  The framework's block rule, as in
    // the MXFP8 GEMM's epilogue: NaN does not enter the block's amax; columns past N are
    // zeros or NaN.
    __device__ __forceinline__ void store_mx(int64_t row, float v) const
    {
        const uint32_t mag = __float_as_uint(v) & 0x7FFFFFFFu;
        const uint32_t amax = __reduce_max_sync(0xFFFFFFFFu, mag > 0x7F800000u ? 0u : mag);
        float inv;
        const uint32_t s = mx_block_scale(__uint_as_float(amax), inv);
        const float q = v * inv;
        if (ok) p.D[row * p.ldd + n] = (uint8_t)f32x2_to_e4m3x2(q, q);
        if ((n & 31) == 0 && ok) p.D_scales[row * p.nblkN + n / 32] = (uint8_t)s;
    }

    // The MX blocks of `count` rows, raw[i] being this column's sum in row row0 + i.  A block's
    // amax and scale are the work of one lane: the warp turns its 32 x 32 sums in shared
    // memory (rows kTurnStride floats apart: reads and writes free of bank conflicts), so
    // that lane i holds row i.
    __device__ __forceinline__ void store_mx_rows(const uint32_t (&raw)[32], int count, int64_t row0, float* turn) const
    {
        const int lane = threadIdx.x & 31;
        __syncwarp();  // the previous chunk has been read
#pragma unroll
        for (int i = 0; i < 32; ++i) turn[i * kTurnStride + lane] = __uint_as_float(raw[i]);
        __syncwarp();
        const int col0 = n - lane, valid = min(32, p.N - col0);
        const bool whole = valid == 32 && p.d_vec;
        float v[32], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float4 q = *reinterpret_cast<const float4*>(turn + lane * kTurnStride + i);
            v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(v[i]));
        float inv;
        const uint32_t s = mx_block_scale(amax, inv);
        uint4 w[2];
        const uint2 q0 = quantize8(v, inv), q1 = quantize8(v + 8, inv);
        const uint2 q2 = quantize8(v + 16, inv), q3 = quantize8(v + 24, inv);
        w[0] = make_uint4(q0.x, q0.y, q1.x, q1.y);
        w[1] = make_uint4(q2.x, q2.y, q3.x, q3.y);
        uint8_t* dst = p.D + (row0 + lane) * p.ldd + col0;
        if (lane < count) {
            p.D_scales[(row0 + lane) * p.nblkN + col0 / 32] = (uint8_t)s;
            if (whole) {
                reinterpret_cast<uint4*>(dst)[0] = w[0];
                reinterpret_cast<uint4*>(dst)[1] = w[1];
            }
        }
        if (whole) return;
        // Ragged or unaligned rows: turned back, so that the warp stores one row at a time.
        __syncwarp();
        uint4* mine = reinterpret_cast<uint4*>(turn + lane * kTurnStride);
        mine[0] = w[0];
        mine[1] = w[1];
        __syncwarp();
        if (lane >= valid) return;
        uint8_t* to = p.D + row0 * p.ldd + n;
        for (int i = 0; i < count; ++i, to += p.ldd)
            *to = reinterpret_cast<const uint8_t*>(turn + i * kTurnStride)[lane];
    }

    template <int kType>
    __device__ __forceinline__ static void put(uint8_t* at, float v)
    {
        if constexpr (kType == MPK_TYPE_F32) *reinterpret_cast<float*>(at) = v;
        else if constexpr (kType == MPK_TYPE_BF16) *reinterpret_cast<__nv_bfloat16*>(at) = __float2bfloat16_rn(v);
        else *reinterpret_cast<__half*>(at) = __float2half_rn(v);
    }

    template <int kType>
    __device__ __forceinline__ static uint32_t pack(float lo, float hi)
    {
        uint32_t r;
        if constexpr (kType == MPK_TYPE_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }

    // `count` rows of this column, `at` the first one's element and `step` bytes between
    // them; sa: the rows' scales in shared memory (int8).  Warp-uniform in count.
    // Whole chunks of a 16-bit D: neighbouring lanes swap halves of two rows' packed values,
    // so that the even lane stores the upper row's two columns and the odd lane the lower
    // row's, 4 bytes each.  Half the stores of one element at a time, which they were bound
    // by (32 rows x 32 columns BF16: 674 clocks that way).
    template <int kType>
    __device__ __forceinline__ void store_rows(const uint32_t (&raw)[32], int count, uint8_t* at, int64_t step,
                                               const float* sa) const
    {
        const int lane = threadIdx.x & 31;
        if (kType != MPK_TYPE_F32 && count == 32 && p.d_vec && n - lane + 32 <= p.N) {
            const uint32_t pick = (lane & 1) != 0 ? 0x3276u : 0x5410u;
            uint8_t* to = (lane & 1) != 0 ? at - 2 + step : at;
            const int64_t two = 2 * step;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if constexpr (C::kInt8) s = *reinterpret_cast<const float4*>(sa + i);
                const uint32_t a = pack<kType>(value(raw[i + 0], s.x), value(raw[i + 1], s.y));
                const uint32_t b = pack<kType>(value(raw[i + 2], s.z), value(raw[i + 3], s.w));
                *reinterpret_cast<uint32_t*>(to) = __byte_perm(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1), pick);
                to += two;
                *reinterpret_cast<uint32_t*>(to) = __byte_perm(b, __shfl_xor_sync(0xFFFFFFFFu, b, 1), pick);
                to += two;
            }
            return;
        }
        if (!ok) return;
        if (count == 32) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if constexpr (C::kInt8) s = *reinterpret_cast<const float4*>(sa + i);
                put<kType>(at + (i + 0) * step, value(raw[i + 0], s.x));
                put<kType>(at + (i + 1) * step, value(raw[i + 1], s.y));
                put<kType>(at + (i + 2) * step, value(raw[i + 2], s.z));
                put<kType>(at + (i + 3) * step, value(raw[i + 3], s.w));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i < count) put<kType>(at + i * step, value(raw[i], C::kInt8 ? sa[i] : 0.0f));
        }
    }
};

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
               const __grid_constant__ CUtensorMap tmap_q16, const Params p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    uint8_t* codes = smem + p.ring_bytes;  // fused quantizer
    uint8_t* control = codes + (C::kFuse ? p.codes_bytes : 0);
    const uint32_t bar0 = smem_u32(control);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
    auto tail = [&](int s) { return bar0 + 8u * (2 * kMaxStages + s); };
    auto tfull = [&](int a) { return bar0 + 8u * (3 * kMaxStages + a); };
    auto tempty = [&](int a) { return bar0 + 8u * (3 * kMaxStages + 2 + a); };
    const uint32_t drain = bar0 + 8u * (3 * kMaxStages + 4);
    const uint32_t codes_ready = bar0 + 8u * (3 * kMaxStages + 5);
    float* tile_scales = reinterpret_cast<float*>(control + kScaleOffset);
    uint32_t* amax_bits = reinterpret_cast<uint32_t*>(control + kCodesOffset);
    float* fused_scales = reinterpret_cast<float*>(amax_bits + kFusedRows);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(control + kMiscOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(control + kMiscOffset + 4);
    volatile int* never_abort = reinterpret_cast<volatile int*>(control + kMiscOffset + 8);
    int* scratch = reinterpret_cast<int*>(control + kMiscOffset + 16);
    int* t_lo = reinterpret_cast<int*>(control + kTableOffset);
    int* t_hi = t_lo + p.E;
    int* t_first = t_hi + p.E;
    const Table tab{t_lo, t_hi, t_first};

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const bool clustered = C::kPair || p.splits > 1;
    const int ctas = C::kCtas * p.splits;  // of a cluster
    const int crank = clustered ? (int)cluster_ctarank() : 0;
    const uint32_t rank = C::kPair ? (uint32_t)(crank & 1) : 0u;  // of the pair
    const int split = crank / C::kCtas;
    const uint32_t leader = (uint32_t)(crank - (int)rank);
    const int unit = (int)blockIdx.x / ctas;
    // Splits: one tile per cluster, whatever the groups say (the host counted tiles of groups
    // that do not overlap, and only one accumulator is allocated).
    const int nunits = p.splits > 1 ? 1 << 30 : (int)gridDim.x / ctas;

    if (warp == 0) {
        if (lane < kMaxStages) {
            mbar_init(full(lane), C::kFullArrivals);
            mbar_init(empty(lane), 1);
            mbar_init(tail(lane), 1);
        } else if (lane < kMaxStages + 2) {
            mbar_init(tfull(lane - kMaxStages), 1);
            mbar_init(tempty(lane - kMaxStages), C::kCtas * C::kEpiWarps);
        } else if (lane == kMaxStages + 2) {
            mbar_init(drain, 1);
            mbar_init(codes_ready, 1);
            *abort_flag = 0;
            *never_abort = 0;
        }
        fence_mbar_init();
    } else if (warp == 3 && p.have_operands) {
        if (lane == 0) prefetch_tmap(&tmap_p);
        if (lane == 1 && !C::kFuse) prefetch_tmap(&tmap_q);
        if (lane == 2 && !C::kWgrad && !C::kFuse) prefetch_tmap(&tmap_q16);
    }
    if (warp == 1) {
        if constexpr (C::kPair) {
            tmem_alloc_pair(smem_u32(tmem_holder), p.tmem_cols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_holder), p.tmem_cols);
            tmem_relinquish();
        }
    }
    int* widest = reinterpret_cast<int*>(control + kMiscOffset + 12);
    // Launched to start while the kernel in front of it still runs: nothing global is touched
    // before that one has completed, except what it is known not to write (p.early).  The
    // next kernel may start likewise, on the SMs that this one's blocks leave first.
    allow_dependent_launch();
    if (!p.early) wait_for_prerequisite_grid();
    build_table<C>(p, t_lo, t_hi, t_first, scratch, widest);
    tc_fence_before();
    __syncthreads();
    if (clustered) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    const int slot_bytes = C::kWgrad ? stage_bytes<C>(kMaxRows) : stage_bytes<C>(*widest);
    const int S = min(kMaxStages, p.ring_bytes / slot_bytes);
    bool producer_aborted = false;
    Walk<C> walk(unit, nunits);
    Tile x = {};
    auto commit = [&](uint32_t bar) {  // arrive on the barrier in the CTAs of this pair
        if constexpr (C::kPair) umma_commit_pair_mc(bar, (uint16_t)(0x3u << leader));
        else umma_commit(bar);
    };

    if (warp == 0) {
        // ------------------------------ TMA producer -------------------------------
        if (elect_one()) {
            const uint64_t policy = p.read_once ? l2_evict_first() : 0u;
            int s = 0, issued = 0;
            uint32_t ph = 0;
            uint32_t last_tail = 0, tail_ph = 0;  // per stage: its last use went through tail(s); uses so, mod 2
            bool ok = true;
            auto load_p = [&](int slot, uint32_t bar, int k) {
                const uint32_t dst = sbase + slot * slot_bytes;
                const int n = x.n0 + kCols * (int)rank;
                auto load = [&](uint32_t to, int c0, int c1, int c2) {
                    if constexpr (C::kPair) tma_load_3d_pair(to, &tmap_p, bar, c0, c1, c2, policy);
                    else tma_load_3d(to, &tmap_p, bar, c0, c1, c2, policy);
                };
                if constexpr (C::kPMn) {
#pragma unroll
                    for (int j = 0; j < kCols / C::kMnBox; ++j)
                        load(dst + j * C::kBoxBytes, n + j * C::kMnBox, C::kWgrad ? x.lo + k : k, C::kWgrad ? 0 : x.e);
                } else {
                    load(dst, k, n, x.e);
                }
            };
            auto load_q = [&](int slot, uint32_t bar, int k) {
                const uint32_t dst = sbase + slot * slot_bytes + P_BYTES;
                const int mine = x.width / C::kCtas;  // rows of this CTA
                const int r = x.r0 + mine * (int)rank;
                auto load = [&](uint32_t to, const CUtensorMap* map, int c0, int c1) {
                    if constexpr (C::kPair) tma_load_2d_pair(to, map, bar, c0, c1);
                    else tma_load_2d(to, map, bar, c0, c1);
                };
                if constexpr (C::kWgrad) {
#pragma unroll
                    for (int j = 0; j < kMaxRows / C::kCtas / C::kMnBox; ++j)
                        load(dst + j * C::kBoxBytes, &tmap_q, r + j * C::kMnBox, x.lo + k);
                } else {
                    int i = 0;
                    for (; i + 64 <= mine; i += 64) load(dst + i * kRowBytes, &tmap_q, k, x.lo + r + i);
                    for (; i < mine; i += 16) load(dst + i * kRowBytes, &tmap_q16, k, x.lo + r + i);
                }
            };
            // A quantizer or pre-pass in front (p.early) makes Q, never P or the groups: the
            // first stages' P loads run under it.
            const bool have = walk.next(p, tab, x);
            int k0 = 0, k1 = 0, early = 0;
            if (have) walk.stages(p, x, split, k0, k1);
            if (!C::kWgrad && have && p.early) {
                early = min(S, k1 - k0);
                for (int i = 0; i < early; ++i) {
                    if (rank == 0)
                        mbar_arrive_expect_tx(full(i), C::kCtas * (uint32_t)stage_bytes<C>(x.width));
                    load_p(i, C::kPair ? mapa_shared(full(i), leader) : full(i), (k0 + i) * C::BK);
                }
            }
            wait_for_prerequisite_grid();
            for (bool more = have; ok && more; more = walk.next(p, tab, x)) {
                walk.stages(p, x, split, k0, k1);
                const int tail_rows = walk.tail_rows(x);
                const uint32_t bytes = (uint32_t)stage_bytes<C>(x.width);
                for (int kb = k0; kb < k1; ++kb) {
                    if (!mbar_wait(empty(s), ph ^ 1u, abort_flag, p.status, kSiteEmpty, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    uint32_t bar;
                    last_tail &= ~(1u << s);
                    if (C::kWgrad && tail_rows > 0 && kb == walk.all_stages(p, x) - 1) {
                        // This CTA's tail warp takes the stage first.
                        bar = tail(s);
                        last_tail |= 1u << s;
                        tail_ph ^= 1u << s;
                        mbar_arrive_expect_tx(bar, bytes);
                        if constexpr (C::kPair) bar = mapa_shared(bar, leader + rank);
                    } else {
                        if (rank == 0 && early == 0) {
                            mbar_arrive_expect_tx(full(s), C::kCtas * bytes);
                            if (C::kFullArrivals == 2) mbar_arrive(full(s));
                        }
                        bar = full(s);
                        if constexpr (C::kPair) bar = mapa_shared(bar, leader);
                    }
                    if (early > 0) --early;
                    else load_p(s, bar, kb * C::BK);
                    if (!C::kFuse) load_q(s, bar, kb * C::BK);
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
        if (rank == 0 && elect_one()) {
            int s = 0, it = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (; ok && walk.next(p, tab, x); ++it) {
                int k0, k1;
                walk.stages(p, x, split, k0, k1);
                const int acc = it & 1;
                if (!mbar_wait(tempty(acc), ((uint32_t)(it >> 1) & 1u) ^ 1u, abort_flag, p.status, kSiteTmemEmpty,
                               p.timeout_ns)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(acc * p.acc_cols);
                const uint32_t idesc = p.idesc | ((uint32_t)(x.width >> 3) << 17);
                const int rem = (x.hi - x.lo) % C::BK;
                if (C::kFuse && it == 0 && !mbar_wait(codes_ready, 0, abort_flag, p.status, kSiteCodes, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                for (int kb = k0; kb < k1; ++kb) {
                    if (!mbar_wait(full(s), ph, abort_flag, p.status, kSiteFull, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    int steps = 4;
                    if (C::kWgrad && rem != 0 && kb == walk.all_stages(p, x) - 1) {
                        steps = (rem + 15) / 16;
                        fence_acq_rel_cluster();  // the tail warps' zeros, of both CTAs
                    }
                    tc_fence_after();
                    const uint32_t a = sbase + s * slot_bytes;
                    const uint32_t b = C::kFuse ? smem_u32(codes) + (kb - k0) * (kFusedRows * kRowBytes) : a + P_BYTES;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (C::kWgrad && k >= steps) break;
                        // A step is 32 bytes along a K-major row, or BK / 4 rows of an MN-major box.
                        constexpr uint32_t kMnStep = C::BK / 4 * kRowBytes;
                        const uint64_t ad = C::kPMn ? umma_smem_desc_sw128(a + k * kMnStep, C::kBoxBytes, 1024)
                                                    : umma_smem_desc_sw128(a + k * 32, 16, 1024);
                        const uint64_t bd = C::kWgrad ? umma_smem_desc_sw128(b + k * kMnStep, C::kBoxBytes, 1024)
                                                      : umma_smem_desc_sw128(b + k * 32, 16, 1024);
                        mma<C>(d, ad, bd, idesc, (kb != k0 || k != 0) ? 1u : 0u);
                    }
                    commit(empty(s));
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                if (!ok) break;
                commit(tfull(acc));
            }
            if constexpr (C::kPair) umma_commit_pair(drain);
            else umma_commit(drain);
            mbar_wait(drain, 0, never_abort, nullptr, 0, kDrainTimeoutNs);
        }
    } else if (C::kWgrad && warp == 2) {
        // ------- tail rows: zeros behind the group's end, in P and in Q -------
        // A zero in one operand alone would leave NaN where the next group's other holds NaN.
        int s = 0;
        uint32_t phases = 0;  // parity of each stage's tail barrier
        const uint32_t full0 = C::kPair ? mapa_shared(full(0), leader) : full(0);
        bool ok = true;
        while (ok && walk.next(p, tab, x)) {
            int k0, k1;
            walk.stages(p, x, split, k0, k1);
            const int rows = k1 == walk.all_stages(p, x) ? walk.tail_rows(x) : 0;  // another split has the last stage
            if (k1 == k0) continue;
            const int last = (s + k1 - k0 - 1) % S;
            s = (last + 1) % S;
            if (rows == 0) continue;
            ok = mbar_wait_warp(tail(last), (phases >> last) & 1u, abort_flag, p.status, kSiteTail, p.timeout_ns);
            if (!ok) break;
            phases ^= 1u << last;
            const int end = (rows + 15) / 16 * 16;
            // 128-byte rows of each box: the swizzle permutes within a row, so whole rows are plain.
            constexpr int kBoxes = (kCols + kMaxRows / C::kCtas) / C::kMnBox;
            const int chunks = (end - rows) * 8;
            for (int j = 0; j < kBoxes; ++j) {
                uint8_t* box = smem + last * slot_bytes + j * C::kBoxBytes;
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
        // The warps of a quarter of the columns take turns at chunks of 32 rows.
        const int quad = warp & 3;
        const int turn = (warp - kFirstEpiWarp) / 4;
        const uint32_t tempty0 = C::kPair ? mapa_shared(tempty(0), leader) : tempty(0);
        float* row_scales = tile_scales + (warp - kFirstEpiWarp) * 32;
        wait_for_prerequisite_grid();  // a_scales may come from the kernel in front
        if constexpr (C::kFuse) {
            Walk<C> first(unit, nunits);
            if (first.next(p, tab, x)) {
                int k0, k1;
                first.stages(p, x, split, k0, k1);
                const int kf = k0 * C::BK, kl = min(p.K, k1 * C::BK), ew = warp - kFirstEpiWarp;
                if (p.x_type == MPK_TYPE_BF16)
                    make_codes<int8::Bf16>(p, ew, lane, kf, kl, codes, amax_bits, fused_scales);
                else if (p.x_type == MPK_TYPE_F16)
                    make_codes<int8::F16>(p, ew, lane, kf, kl, codes, amax_bits, fused_scales);
                else
                    make_codes<int8::F32>(p, ew, lane, kf, kl, codes, amax_bits, fused_scales);
                if (ew == 0 && lane == 0) mbar_arrive(codes_ready);
            }
        }
        // A cluster of splits has one tile, joined below.
        for (int it = 0; p.splits == 1 && walk.next(p, tab, x); ++it) {
            const int acc = it & 1;
            const Column<C> col(p, x, x.n0 + kCols * (int)rank + quad * 32 + lane);
            const bool warp_ok = col.n - lane < p.N;
            int k0, k1;
            walk.stages(p, x, split, k0, k1);
            const bool any = k1 > k0;  // otherwise nothing was accumulated: zeros
            const int64_t row0 = C::kWgrad ? (int64_t)x.r0 : (int64_t)x.lo + x.r0;
            const int64_t base0 = (C::kWgrad ? x.e * p.d_group : 0) + row0 * p.ldd;
            float sa[4];  // scale of this lane's row of each chunk, loaded under the MMAs
            if constexpr (C::kInt8) {
                static_assert(!C::kInt8 || 4 * 32 * C::kTurns == kMaxRows, "four chunks per warp");
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 32 * (C::kTurns * j + turn) + lane;
                    sa[j] = r < x.rows ? (C::kFuse ? fused_scales[r & (kFusedRows - 1)] : p.a_scales[row0 + r]) : 0.0f;
                }
            }
            if (!mbar_wait_warp(tfull(acc), (uint32_t)(it >> 1) & 1u, abort_flag, p.status, kSiteTmemFull,
                                p.timeout_ns))
                break;
            tc_fence_after();
            const uint32_t tacc = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * p.acc_cols);
            if (warp_ok) {
                int j = 0;
#pragma unroll 1
                for (int c = 32 * turn; c < x.rows; c += 32 * C::kTurns, ++j) {
                    __syncwarp();  // lanes past N leave a chunk's stores early; the load takes the whole warp
                    uint32_t raw[32];
                    if (any) {
                        tmem_ld_32x32b_x32(tacc + (uint32_t)c, raw);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) raw[i] = 0u;
                    }
                    const int count = min(32, x.rows - c);
                    if constexpr (C::kMx) {
                        col.store_mx_rows(raw, count, row0 + c,
                                          reinterpret_cast<float*>(control + p.parts_offset) +
                                              (warp - kFirstEpiWarp) * 32 * kTurnStride);
                    } else {
                        if constexpr (C::kInt8) {
                            __syncwarp();
                            row_scales[lane] = j == 0 ? sa[0] : j == 1 ? sa[1] : j == 2 ? sa[2] : sa[3];
                            __syncwarp();
                        }
                        const int eb = p.d_type == MPK_TYPE_F32 ? 4 : 2;
                        uint8_t* at = p.D + (base0 + c * p.ldd + col.n) * eb;
                        const int64_t step = p.ldd * eb;
                        if (p.d_type == MPK_TYPE_BF16)
                            col.template store_rows<MPK_TYPE_BF16>(raw, count, at, step, row_scales);
                        else if (p.d_type == MPK_TYPE_F16)
                            col.template store_rows<MPK_TYPE_F16>(raw, count, at, step, row_scales);
                        else
                            col.template store_rows<MPK_TYPE_F32>(raw, count, at, step, row_scales);
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
    __syncwarp();

    if (p.splits > 1 && unit < tab.first[p.E]) {
        // Join the splits' sums in their order.  Block g of four rows is finished by split
        // g % splits: every CTA hands its part of the block to that split's CTA of the same
        // columns, as block g / splits of slice `split` there ([block][column][4 rows]).
        Walk<C> again(unit, nunits);
        again.next(p, tab, x);
        const int ew = warp - kFirstEpiWarp;
        const int quad = warp & 3, turn = ew / 4;
        const int blocks = (x.rows + 3) / 4, share = (blocks + p.splits - 1) / p.splits;
        const int64_t row0 = C::kWgrad ? (int64_t)x.r0 : (int64_t)x.lo + x.r0;
        const int64_t base0 = C::kWgrad ? x.e * p.d_group : 0;
        int k0, k1;
        again.stages(p, x, split, k0, k1);  // a short group may leave this split nothing
        const Column<C> col(p, x, x.n0 + kCols * (int)rank + quad * 32 + lane);
        const bool busy = ew >= 0 && col.n - lane < p.N;
        // Slices lie in the ring's place if there is no room behind it: then every CTA's
        // MMAs must be done before the first block arrives.
        uint8_t* parts = p.parts_in_ring ? smem : control + p.parts_offset;
        bool ok = true;
        if (ew >= 0) {
            if (C::kInt8) {
                const int r = ew * 32 + lane;
                if (r < x.rows) tile_scales[r] = C::kFuse ? fused_scales[r & (kFusedRows - 1)] : p.a_scales[row0 + r];
            }
            ok = mbar_wait_warp(tfull(0), 0, abort_flag, p.status, kSiteTmemFull, p.timeout_ns);
            // A part that never came must not be added: the whole cluster stores nothing.  The
            // barrier below makes the flags visible before any CTA looks at its own.
            if (!ok && lane < ctas)
                st_shared_cluster_u32(mapa_shared(smem_u32(const_cast<int*>(abort_flag)), (uint32_t)lane), 1u);
            tc_fence_after();
        }
        __syncwarp();  // columns past N loaded no scales; the barriers take whole warps
        if (p.parts_in_ring) cluster_sync_all();
        if (busy && ok) {
            const uint32_t tacc = tmem_base + ((uint32_t)(quad * 32) << 16);
            const uint32_t mine = smem_u32(parts) + 16u * (uint32_t)(split * share * kCols + quad * 32 + lane);
#pragma unroll 1
            for (int c = 32 * turn; c < x.rows; c += 32 * C::kTurns) {
                __syncwarp();
                uint32_t raw[32];
                if (k1 > k0) {
                    tmem_ld_32x32b_x32(tacc + (uint32_t)c, raw);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) raw[i] = 0u;
                }
                int to = (c / 4) % p.splits, block = (c / 4) / p.splits;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    if (c + i < x.rows)
                        st_shared_cluster_v4(mapa_shared(mine + 16u * (uint32_t)(block * kCols),
                                                         (uint32_t)(to * C::kCtas) + rank),
                                             make_uint4(raw[i], raw[i + 1], raw[i + 2], raw[i + 3]));
                    if (++to == p.splits) to = 0, ++block;
                }
            }
        }
        __syncwarp();
        cluster_sync_all();
        if (busy && *abort_flag == 0) {
            const uint4* part = reinterpret_cast<const uint4*>(parts) + quad * 32 + lane;
            for (int j = turn; split + j * p.splits < blocks; j += C::kTurns) {
                uint4 v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < p.splits) v[q] = part[(q * share + j) * kCols];
                uint32_t sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
                for (int q = 1; q < 8; ++q) {
                    if (q >= p.splits) break;
                    const uint32_t w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sum[i] = C::kInt8 ? sum[i] + w[i]
                                          : __float_as_uint(__uint_as_float(sum[i]) + __uint_as_float(w[i]));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * (split + j * p.splits) + i;
                    if (r >= x.rows) break;
                    const int64_t row = row0 + r;
                    const float d = col.value(sum[i], C::kInt8 ? tile_scales[r] : 0.0f);
                    if constexpr (C::kMx) {
                        col.store_mx(row, d);
                    } else if (col.ok) {
                        uint8_t* at = p.D + (base0 + row * p.ldd + col.n) * (p.d_type == MPK_TYPE_F32 ? 4 : 2);
                        if (p.d_type == MPK_TYPE_BF16) col.template put<MPK_TYPE_BF16>(at, d);
                        else if (p.d_type == MPK_TYPE_F16) col.template put<MPK_TYPE_F16>(at, d);
                        else col.template put<MPK_TYPE_F32>(at, d);
                    }
                }
            }
        }
        __syncwarp();
    }

    if (producer_aborted) {
        // A copy of the other CTA may still be landing after rank 0 stopped expecting it.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 100000ull) {
        }
    }
    __syncwarp();
    tc_fence_before();
    if (clustered) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (C::kPair) tmem_dealloc_pair(tmem_base, p.tmem_cols);
        else tmem_dealloc(tmem_base, p.tmem_cols);
    }
}

// MXFP8 rows -> BF16 rows padded to a multiple of 8 elements, for a K or an alignment that the
// codec's kernel takes element by element: a warp per row, 8 codes per lane and step from
// two aligned 8-byte words (the granules that hold them lie within the codes).
constexpr int kUnpackThreads = 256;

__global__ void __launch_bounds__(kUnpackThreads)
mxfp8_unpack_rows_kernel(const uint8_t* data, const uint8_t* scales, uint16_t* out, int64_t M, int64_t K, int64_t ld_out)
{
    wait_for_prerequisite_grid();
    allow_dependent_launch();
    const int lane = threadIdx.x & 31;
    const int64_t nblk = (K + 31) / 32, warps = (int64_t)gridDim.x * (kUnpackThreads / 32);
    for (int64_t m = (int64_t)blockIdx.x * (kUnpackThreads / 32) + threadIdx.x / 32; m < M; m += warps) {
        const uint8_t* row = data + m * K;
        for (int64_t k = 8 * lane; k < K; k += 256) {
            const uint8_t* at = row + k;
            const uint8_t* word = at - (reinterpret_cast<uintptr_t>(at) & 7u);
            const int shift = 8 * (int)(at - word);
            uint64_t c;
            if (k + 8 <= K && word >= data && word + 16 <= data + M * K) {
                c = load_8b(word);
                if (shift != 0)
                    c = (c >> shift) | (load_8b(word + 8) << (64 - shift));
            } else {
                c = 0u;
                for (int j = 0; j < 8 && k + j < K; ++j) c |= (uint64_t)row[k + j] << (8 * j);
            }
            const float s = e8m0_to_f32(scales[m * nblk + k / 32]);
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = e4m3x2_to_f32x2((uint32_t)(c >> (16 * j)) & 0xFFFFu);
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(f.y * s), "f"(f.x * s));
            }
            *reinterpret_cast<uint4*>(out + m * ld_out + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

}  // namespace product

// ----------------------------------------------------------------------------
// Host side
// ----------------------------------------------------------------------------
namespace {

std::mutex g_attr_mu;
constexpr int kSmemMax = 232448;  // of one block

int pow2_at_least(int x)
{
    int p = 32;
    while (p < x) p *= 2;
    return p;
}

template <class C>
int launch_config(const ProductArgs& a, product::Params& p, cudaStream_t stream, int dev)
{
    using namespace product;
    static bool attr_set[64] = {};
    static int max_clusters[64][9] = {};  // [device][CTAs of a cluster], 0: not asked yet
    const int eb = C::kInt8 ? 1 : 2;
    CUtensorMap tp{}, tq{}, tq16{};
    const CUtensorMapDataType dt = C::kInt8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : a.ab_type == MPK_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int reduction = C::kWgrad ? a.M : a.K;
    p.have_operands = reduction > 0;
    if (reduction > 0) {  // otherwise no load is issued
        const uint64_t qdims[2] = {(uint64_t)a.K, (uint64_t)a.M};
        const uint64_t qstr[1] = {(uint64_t)a.lda * eb};
        const uint32_t qbox[2] = {(uint32_t)(C::kWgrad ? C::kMnBox : C::BK), 64u};
        if (!C::kFuse) {
            if (int rc = encode_tensor_map(&tq, dt, a.A, 2, qdims, qstr, qbox)) return rc;
        }
        if (!C::kWgrad && !C::kFuse) {
            const uint32_t qbox16[2] = {(uint32_t)C::BK, 16u};
            if (int rc = encode_tensor_map(&tq16, dt, a.A, 2, qdims, qstr, qbox16)) return rc;
        }
        const int p_inner = C::kPMn ? a.N : a.K;
        const int p_rows = C::kWgrad ? a.M : (C::kPMn ? a.K : a.N);
        const uint64_t pdims[3] = {(uint64_t)p_inner, (uint64_t)p_rows, (uint64_t)(C::kWgrad ? 1 : a.E)};
        const uint64_t pstr[2] = {(uint64_t)a.ldb * eb, (uint64_t)a.ldb * eb * (uint64_t)p_rows};
        const uint32_t pbox[3] = {(uint32_t)(C::kPMn ? C::kMnBox : C::BK), (uint32_t)(C::kPMn ? C::BK : kCols), 1u};
        if (int rc = encode_tensor_map(&tp, dt, a.B, 3, pdims, pstr, pbox)) return rc;
    }
    p.num_kb = (a.K + C::BK - 1) / C::BK;
    p.num_n_tiles = (a.N + kCols * C::kCtas - 1) / (kCols * C::kCtas);
    if (C::kInt8)
        p.idesc = (2u << 4) | (1u << 7) | (1u << 10);  // S32 sums, signed 8-bit operands
    else
        p.idesc = (1u << 4) | (a.ab_type == MPK_TYPE_BF16 ? (1u << 7) | (1u << 10) : 0u);  // FP32 sums
    p.idesc |= ((C::kPMn ? 1u : 0u) << 15) | ((C::kWgrad ? 1u : 0u) << 16) |
               ((uint32_t)(kCols * C::kCtas >> 4) << 24);

    // At most this many tiles (a group of r rows has ceil(r / kMaxRows) row tiles); the
    // walk counts them in 32 bits.
    const int64_t row_tiles = C::kWgrad ? (int64_t)a.E * ((a.K + kMaxRows - 1) / kMaxRows)
                                        : (int64_t)a.M / kMaxRows + std::min(a.E, a.M);
    const int64_t tiles = row_tiles * p.num_n_tiles;
    // Nor may groups that overlap, against the rules, count past 32 bits.
    const int64_t most_tiles = C::kWgrad ? tiles : (int64_t)a.E * ((a.M + (int64_t)kMaxRows - 1) / kMaxRows) * p.num_n_tiles;
    if (tiles > INT32_MAX / 16 || most_tiles > INT32_MAX / 2) {
        set_last_error("product of too many tiles (M=%d N=%d K=%d, %d groups)", a.M, a.N, a.K, a.E);
        return MPK_ERR_UNSUPPORTED;
    }
    const int64_t units = device_sm_count() / C::kCtas;  // tiles at once
    const int rows = C::kWgrad ? kMaxRows
                               : std::min(kMaxRows, (a.M + C::kRowStep - 1) / C::kRowStep * C::kRowStep);
    const auto kernel = product_kernel<C>;
    std::unique_lock<std::mutex> lk(g_attr_mu);
    if (!attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
        if (e != cudaSuccess) {
            set_last_error("cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
            return (int)e;
        }
        attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    const auto set_cluster = [&](int ctas) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)ctas;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = ctas > 1 ? 1 : 0;
    };
    // Fewer tiles than SMs: share each tile's reduction among the CTAs of a cluster, of
    // at most 8 CTAs, each with at least 4 stages of it, if all clusters can run at once.
    p.splits = 1;
    if (2 * tiles <= units) {
        const int64_t stages = C::kWgrad ? (int64_t)a.M / a.E / C::BK : p.num_kb;
        int most = (int)std::min<int64_t>({units / tiles, 8 / C::kCtas, stages / 4});
        for (; most > 1; --most) {
            const int ctas = C::kCtas * most;
            int& n = max_clusters[dev][ctas];
            if (n == 0) {
                set_cluster(ctas);
                cfg.gridDim = dim3((unsigned)ctas, 1, 1);
                cfg.dynamicSmemBytes = (size_t)kSmemMax;
                if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                    cudaGetLastError();
                    n = 0;
                    most = 1;
                    break;
                }
            }
            if (n >= tiles) break;
        }
        p.splits = std::max(most, 1);
    }
    lk.unlock();
    p.acc_cols = pow2_at_least(rows);
    p.tmem_cols = p.splits > 1 ? p.acc_cols : 2 * p.acc_cols;
    p.codes_bytes = C::kFuse ? (p.num_kb + p.splits - 1) / p.splits * kFusedRows * kRowBytes : 0;
    // Splits join a tile's sums in shared memory: up to 32 KiB behind the ring, else in the
    // ring's place.  They take splits * ceil(rows / 4 / splits) * 2048 bytes, at most
    // 142 KiB, and a ring that fills the SM's shared memory has 160 KiB.
    const int parts = p.splits > 1 ? ((rows + 3) / 4 + p.splits - 1) / p.splits * p.splits * 4 * kCols * 4 : 0;
    p.parts_in_ring = parts > 32768;
    p.parts_offset = (control_bytes(a.E) + 15) / 16 * 16;
    const int turn = C::kMx && p.splits == 1 ? C::kEpiWarps * 32 * kTurnStride * 4 : 0;
    const int behind = p.codes_bytes + p.parts_offset + (p.parts_in_ring ? 0 : parts) + turn + 1024;
    p.ring_bytes = std::min(kMaxStages * stage_bytes<C>(rows), (kSmemMax - behind) / 1024 * 1024);
    const int ctas = C::kCtas * p.splits;
    const int64_t grid = p.splits > 1 ? tiles : std::min(tiles, units);
    cfg.gridDim = dim3((unsigned)(grid * ctas), 1, 1);
    cfg.dynamicSmemBytes = (size_t)(p.ring_bytes + behind);
    set_cluster(ctas);
    // Where hardly a group has a second row tile, weights that leave L2 first leave room for the
    // rows (16 experts of 2048x4096, 1000 rows: 48.3 -> 45.6 us); at 128 rows per group, a
    // few of them above 256, it costs 3 %.
    p.read_once = !C::kWgrad && (a.E == 1 ? a.M <= kMaxRows : (int64_t)a.M <= 64 * (int64_t)a.E);
    p.early = a.after_kernel;
    if (a.after_kernel || !stream_captures(stream)) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tp, tq, tq16, p);
    if (e == cudaErrorInvalidValue || e == cudaErrorLaunchOutOfResources) {
        // A context re-created by cudaDeviceReset has lost the shared-memory attribute.
        cudaGetLastError();
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax) == cudaSuccess)
            e = cudaLaunchKernelEx(&cfg, kernel, tp, tq, tq16, p);
    }
    if (e != cudaSuccess) {
        set_last_error("product launch failed: %s", cudaGetErrorString(e));
        return (int)e;
    }
    return MPK_SUCCESS;
}

template <bool kInt8, bool kPMn, bool kMx>
int launch_rows(const ProductArgs& a, product::Params& p, cudaStream_t stream, int dev)
{
    using namespace product;
    // A pair's tile has 256 columns and halves the loads of A; single CTAs give twice the
    // tiles, for groups too small for that to matter and for products of few tiles.
    const int64_t row_tiles = (int64_t)a.M / kMaxRows + std::min(a.E, a.M);
    const bool pair = (int64_t)a.M > 48 * (int64_t)a.E && a.N > kCols &&
                      row_tiles * ((a.N + 2 * kCols - 1) / (2 * kCols)) * 4 > device_sm_count();
    if constexpr (kInt8) {
        if (a.x) return launch_config<Config<true, kPMn, false, false, false, true>>(a, p, stream, dev);
    }
    if (pair) return launch_config<Config<kInt8, kPMn, false, true, kMx>>(a, p, stream, dev);
    return launch_config<Config<kInt8, kPMn, false, false, kMx>>(a, p, stream, dev);
}

}  // namespace

cudaError_t launch_mxfp8_unpack_rows(const uint8_t* data, const uint8_t* scales, void* out, int64_t M, int64_t K,
                                     int64_t ld_out, cudaStream_t stream)
{
    using namespace product;
    if (M == 0 || K == 0) return cudaSuccess;
    const int64_t blocks = std::min<int64_t>((M + kUnpackThreads / 32 - 1) / (kUnpackThreads / 32),
                                             (int64_t)device_sm_count() * 8);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kUnpackThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = stream_captures(stream) ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, mxfp8_unpack_rows_kernel, data, scales, static_cast<uint16_t*>(out), M, K, ld_out);
}

// Rows at any address to rows on 16-byte boundaries, for operands that TMA cannot read in
// place.  HBM bound: a thread makes 16-byte pieces of a row from the two aligned pieces that
// hold each (the second is in L1 for its neighbour), shifted together; pieces at the row's ends are
// read by element, so nothing outside the rows is touched.  36000 rows of 3414 BF16: 113 us, 4.3
// TB/s, where cudaMemcpy2DAsync takes 267.
namespace product {
constexpr int kPadThreads = 256, kPadBatch = 4;

template <class T>
__global__ void __launch_bounds__(kPadThreads)
pad_rows_kernel(const T* __restrict__ x, int64_t ldx, T* __restrict__ out, int64_t ld_out, int64_t rows,
                int64_t cols, int across_log2)
{
    constexpr int V = 16 / sizeof(T);
    const int across = 1 << across_log2, per_block = kPadThreads >> across_log2;
    const int tx = threadIdx.x & (across - 1), ty = threadIdx.x >> across_log2;
    const int64_t nvec = (cols + V - 1) / V;
    for (int64_t m = (int64_t)blockIdx.x * per_block + ty; m < rows; m += (int64_t)gridDim.x * per_block) {
        const T* row = x + m * ldx;
        uint4* to = reinterpret_cast<uint4*>(out + m * ld_out);
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row) % 16);  // bytes
        const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) - off);
        const int64_t end = off + cols * (int64_t)sizeof(T);  // of the row, bytes behind `from`
        const auto piece = [&](int64_t j) {
            uint32_t w[8] = {};
            if (off == 0 ? 16 * (j + 1) <= end : j > 0 && 16 * (j + 2) <= end) {
                const uint4 lo = __ldg(from + j);
                w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w;
                if (off != 0) {
                    const uint4 hi = __ldg(from + j + 1);
                    w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
                }
#pragma unroll
                for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
                for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (off & 3));
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (j * V + i < cols)
                        w[i * sizeof(T) / 4] |= (uint32_t)__ldg(row + j * V + i) << (8 * sizeof(T) * i % 32);
            }
            return make_uint4(w[0], w[1], w[2], w[3]);
        };
        for (int64_t j = tx; j < nvec; j += kPadBatch * across) {
            uint4 q[kPadBatch];
#pragma unroll
            for (int u = 0; u < kPadBatch; ++u)
                if (j + u * across < nvec) q[u] = piece(j + u * across);
#pragma unroll
            for (int u = 0; u < kPadBatch; ++u)
                if (j + u * across < nvec) to[j + u * across] = q[u];
        }
    }
}
}  // namespace product

cudaError_t launch_pad_rows(const void* x, int64_t ldx, void* out, int64_t ld_out, int64_t rows, int64_t cols,
                            int elem_bytes, cudaStream_t stream)
{
    using namespace product;
    if (rows == 0 || cols == 0) return cudaSuccess;
    const int64_t nvec = (cols * elem_bytes + 15) / 16;
    // 64 threads across a row (36000 rows of 427 pieces: 113 us, 131 with 256), all of them where
    // rows are too few to give every SM some.
    const int most = rows >= 4 * (int64_t)device_sm_count() ? 64 : kPadThreads;
    int across_log2 = 0;
    while ((1 << across_log2) < most && (1 << across_log2) < nvec) ++across_log2;
    const int per_block = kPadThreads >> across_log2;
    const unsigned blocks = (unsigned)std::min<int64_t>((rows + per_block - 1) / per_block,
                                                        (int64_t)device_sm_count() * 32);
    if (elem_bytes == 1)
        pad_rows_kernel<<<blocks, kPadThreads, 0, stream>>>(static_cast<const uint8_t*>(x), ldx,
                                                            static_cast<uint8_t*>(out), ld_out, rows, cols, across_log2);
    else
        pad_rows_kernel<<<blocks, kPadThreads, 0, stream>>>(static_cast<const uint16_t*>(x), ldx,
                                                            static_cast<uint16_t*>(out), ld_out, rows, cols,
                                                            across_log2);
    return cudaGetLastError();
}

bool stream_captures(cudaStream_t stream)
{
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &status) != cudaSuccess) {
        cudaGetLastError();
        return true;
    }
    return status != cudaStreamCaptureStatusNone;
}

// Few rows are quantized by the product's own CTAs, each for itself, if the codes of their
// whole reduction leave room for the ring.  Every CTA then reads all of x; against the row
// quantizer in front, which costs a launch and a workspace, measured on B200: 1 x 4096 x 4096 9.6
// against 12.3 us, 16 x 512 x 512 7.2 against 8.6; 4 x 12288 x 4096 14.4 against 13.5.
bool product_quantizes(int M, int K)
{
    return M <= product::kFusedRows && K > 0 && (int64_t)M * K <= 8192;
}

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
    p.d_vec = a.d_type == kTypeMxfp8 ? reinterpret_cast<uintptr_t>(a.D) % 16 == 0 && a.ldd % 16 == 0
                                     : reinterpret_cast<uintptr_t>(a.D) % 4 == 0 && a.ldd % 2 == 0;
    p.D_scales = a.D_scales;
    p.nblkN = (a.N + 31) / 32;
    p.a_scales = a.a_scales;
    p.b_scales = a.b_scales;
    p.bias = a.bias;
    p.x = a.x;
    p.ldx = a.ldx;
    p.x_type = a.x_type;
    p.K = a.K;
    p.x_vec = a.x && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx * (a.x_type == MPK_TYPE_F32 ? 4 : 2) % 16 == 0;
    p.status = status;
    p.timeout_ns = wait_timeout_ns();
    if (a.wgrad) return launch_config<Config<false, true, true, true, false>>(a, p, stream, dev);
    if (a.ab_type == kTypeInt8)
        return a.b_nk ? launch_rows<true, false, false>(a, p, stream, dev)
                      : launch_rows<true, true, false>(a, p, stream, dev);
    if (a.d_type == kTypeMxfp8) return launch_rows<false, true, true>(a, p, stream, dev);
    return a.b_nk ? launch_rows<false, false, false>(a, p, stream, dev)
                  : launch_rows<false, true, false>(a, p, stream, dev);
}

}  // namespace mpk
