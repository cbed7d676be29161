// Quantizers to 8-bit integers with one FP32 scale per row (token) or per column
// (output channel of a weight).  HBM bound.
// The numerics are int8_codes.cuh's.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "int8_codes.cuh"
#include "mpk.h"
#include "mpk_internal.h"
#include "mpk_ptx.cuh"

namespace mpk {
namespace {

namespace cg = cooperative_groups;

using namespace int8;

// ------------------------------- rows ---------------------------------------
// kPerRow threads hold a row in registers, up to kHold 16-byte pieces each, all loaded
// before the first is used: one pass over x.  Longer rows are read twice, the second time
// from L1 or L2.  Captured, with other rows each time: 16384 x 2048 BF16 in 22.2 us (4.5 TB/s of
// the least bytes), 4096 x 8192 FP32 in 34.3 us (4.9 TB/s).  Two blocks fit an SM (127 registers),
// and a warp's loads, maximum and stores follow one another: HBM idles at each row's end.
constexpr int kRowThreads = 256, kHold = 16;

template <class D, int kPerRow>
__global__ void __launch_bounds__(kRowThreads)
int8_quantize_rows_kernel(const typename D::T* x, int64_t ldx, int8_t* codes,
                          int64_t ld_codes, float* scales, int64_t M, int64_t K, int)
{
    // Started while the kernel in front may still run.  The product that follows may in turn
    // load its weights once every block is past this wait: nothing in front of this kernel
    // can be writing them then.
    wait_for_prerequisite_grid();
    allow_dependent_launch();
    constexpr int kRows = kRowThreads / kPerRow;  // of a block
    __shared__ uint32_t warp_max[kRowThreads / 32];
    const int tid = threadIdx.x % kPerRow;
    const int64_t nvec = K / D::kVec;
    const bool held = nvec <= (int64_t)kPerRow * kHold;  // the same for every row
    for (int64_t m0 = (int64_t)blockIdx.x * kRows; m0 < M; m0 += (int64_t)gridDim.x * kRows) {
        const int64_t m = m0 + threadIdx.x / kPerRow;
        const bool have = m < M;
        const typename D::T* row = x + (have ? m : 0) * ldx;
        int8_t* out = codes + (have ? m : 0) * ld_codes;
        uint32_t amax = 0;
        uint4 h[kHold];
        if (held) {
#pragma unroll
            for (int j = 0; j < kHold; ++j) {
                if (j * kPerRow >= nvec) break;
                const int64_t i = (int64_t)j * kPerRow + tid;
                h[j] = have && i < nvec ? load_16b(reinterpret_cast<const uint4*>(row) + i) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int j = 0; j < kHold; ++j) {
                if (j * kPerRow >= nvec) break;
                amax = max(amax, largest(D(), h[j]));
            }
        } else if (have) {
            for (int64_t i = tid; i < nvec; i += kPerRow)
                amax = max(amax, largest(D(), load_16b(reinterpret_cast<const uint4*>(row) + i)));
        }
        if (have)
            for (int64_t k = nvec * D::kVec + tid; k < K; k += kPerRow)
                amax = max(amax, magnitude(D::widen(row[k])));
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        if constexpr (kPerRow > 32) {
            if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kRowThreads / 32; ++w) amax = max(amax, warp_max[w]);
        }
        const RowScale rs = row_scale(amax);
        if (have) {
            if (tid == 0) scales[m] = rs.scale;
            const auto put = [&](int64_t i, const uint4& q) {
                float v[D::kVec];
                D::widen(q, v);
                if constexpr (D::kVec == 8)
                    *reinterpret_cast<uint2*>(out + i * 8) = make_uint2(pack4(v, rs.inv), pack4(v + 4, rs.inv));
                else
                    *reinterpret_cast<uint32_t*>(out + i * 4) = pack4(v, rs.inv);
            };
            if (held) {
#pragma unroll
                for (int j = 0; j < kHold; ++j) {
                    if (j * kPerRow >= nvec) break;
                    const int64_t i = (int64_t)j * kPerRow + tid;
                    if (i < nvec) put(i, h[j]);
                }
            } else {
                for (int64_t i = tid; i < nvec; i += kPerRow) put(i, load_16b(reinterpret_cast<const uint4*>(row) + i));
            }
            for (int64_t k = nvec * D::kVec + tid; k < K; k += kPerRow)
                out[k] = rs.inv == 0.0f ? (int8_t)0 : (int8_t)code_bits(D::widen(row[k]), rs.inv);
        }
        if constexpr (kPerRow > 32) __syncthreads();  // warp_max is read before the next row writes it
    }
}

// Rows that do not start on a 16-byte boundary are still read in aligned pieces: piece i
// holds elements i * kVec - off ..., off being the row's distance from the boundary before
// it, and elements outside the row count as zeros.  The codes of piece i and the next one,
// shifted against each other by off bytes, make output word i.  Such rows are read twice,
// a warp each where there are many (8846 x 4991 BF16 in 51 us; 65 us with a block per row).
constexpr int kShiftedBatch = 4;  // pieces in flight per thread

template <class D>
__device__ __forceinline__ uint4 shifted_piece(const typename D::T* row, int64_t k, int64_t K)
{
    if (k >= 0 && k + D::kVec <= K) return load_16b(row + k);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    constexpr int kBits = 8 * sizeof(typename D::T), kPer = 32 / kBits;
#pragma unroll
    for (int j = 0; j < D::kVec; ++j)
        if (k + j >= 0 && k + j < K) {
            uint32_t e;
            if constexpr (sizeof(typename D::T) == 4) e = __float_as_uint(row[k + j]);
            else e = row[k + j];
            w[j / kPer] |= e << (kBits * (j % kPer));
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The codes of a piece, the first in the lowest byte.
template <class D>
__device__ __forceinline__ uint64_t piece_codes(const uint4& q, float inv)
{
    float v[D::kVec];
    D::widen(q, v);
    uint64_t c = pack4(v, inv);
    if constexpr (D::kVec == 8) c |= (uint64_t)pack4(v + 4, inv) << 32;
    return c;
}

template <class D, int kPerRow>
__global__ void __launch_bounds__(kRowThreads)
int8_quantize_shifted_rows_kernel(const typename D::T* x, int64_t ldx, int8_t* codes,
                          int64_t ld_codes, float* scales, int64_t M, int64_t K, int words_ok)
{
    wait_for_prerequisite_grid();
    allow_dependent_launch();
    constexpr int V = D::kVec;
    constexpr int kRows = kRowThreads / kPerRow;  // of a block
    __shared__ uint32_t warp_max[kRowThreads / 32];
    const int tid = threadIdx.x % kPerRow;
    for (int64_t m0 = (int64_t)blockIdx.x * kRows; m0 < M; m0 += (int64_t)gridDim.x * kRows) {
        const int64_t m = m0 + threadIdx.x / kPerRow;
        const bool have = m < M;
        const typename D::T* row = x + (have ? m : 0) * ldx;
        int8_t* out = codes + (have ? m : 0) * ld_codes;
        const int off = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(typename D::T));
        const int64_t nvec = (off + K + V - 1) / V;
        const auto piece = [&](int64_t i) { return shifted_piece<D>(row, i * V - off, K); };
        uint32_t amax = 0;
        if (have) {
            for (int64_t j = tid; j < nvec; j += kShiftedBatch * kPerRow) {
                uint4 q[kShiftedBatch];
#pragma unroll
                for (int u = 0; u < kShiftedBatch; ++u)
                    q[u] = j + u * kPerRow < nvec ? piece(j + u * kPerRow) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int u = 0; u < kShiftedBatch; ++u) amax = max(amax, largest(D(), q[u]));
            }
        }
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        if constexpr (kPerRow > 32) {
            if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = amax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kRowThreads / 32; ++w) amax = max(amax, warp_max[w]);
        }
        const RowScale rs = row_scale(amax);
        if (have && tid == 0) scales[m] = rs.scale;
        // Output word i, the codes of elements i * V .. (V of them, fewer at the row's end); all
        // lanes of a warp call it together.  Words go out whole where the codes' rows allow.
        const auto put = [&](int64_t i, const uint4& q) {
            uint64_t c = piece_codes<D>(q, rs.inv);
            uint64_t next = __shfl_down_sync(0xFFFFFFFFu, c, 1);
            if (off != 0) {
                if ((threadIdx.x & 31) == 31) next = have ? piece_codes<D>(piece(i + 1), rs.inv) : 0u;
                c = (c >> (8 * off)) | (next << (8 * (V - off)));
            }
            const int64_t left = have ? K - i * V : 0;
            if (left <= 0) return;
            if (words_ok && left >= V) {
                if constexpr (V == 8)
                    *reinterpret_cast<uint2*>(out + i * 8) = make_uint2((uint32_t)c, (uint32_t)(c >> 32));
                else
                    *reinterpret_cast<uint32_t*>(out + i * 4) = (uint32_t)c;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j < left) out[i * V + j] = (int8_t)(c >> (8 * j));
            }
        };
        for (int64_t j = tid; j - tid < nvec; j += kShiftedBatch * kPerRow) {  // warp-uniform: put shuffles
            uint4 q[kShiftedBatch];
#pragma unroll
            for (int u = 0; u < kShiftedBatch; ++u)
                q[u] = have && j + u * kPerRow < nvec ? piece(j + u * kPerRow) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int u = 0; u < kShiftedBatch; ++u) put(j + u * kPerRow, q[u]);
        }
        if constexpr (kPerRow > 32) __syncthreads();  // warp_max is read before the next row writes it
    }
}

// ------------------------------ columns -------------------------------------
// A cluster of blocks per strip of columns and expert: each block takes a share of the
// rows, the strip's largest magnitudes are joined through distributed shared memory, and
// a second pass over the share makes the codes.  The second pass finds the share in L2 on
// the block's own side of the chip; two kernels with the maxima in memory between them,
// or a share held in registers or shared memory, took as long or longer (4096 x 12288
// BF16: 37 us, 4.1 TB/s of the least bytes; 44, 52 and 38 us).
constexpr int kColThreads = 256;
constexpr int kColBatch = 8;    // rows a thread has in flight
constexpr int kColBlocks = 3;   // resident blocks per SM
constexpr int kColWide = 16;    // threads across a strip
constexpr int kColCtas = 8;     // most blocks per strip
constexpr int kColShare = 512;  // rows of one of them, where there are strips enough

template <class D, bool kVector, int kAcross>  // kAcross threads across a strip
struct Cols {
    static constexpr int V = kVector ? D::kVec : 1;
    static constexpr int kStrip = kAcross * V;
    static constexpr int kDown = kColThreads / kAcross;  // rows per step
    using Piece = std::conditional_t<kVector, uint4, typename D::T>;
    // use(row, piece) for this thread's rows of [k0, k1), kColBatch loads at a time.
    template <class F>
    static __device__ __forceinline__ void each(const typename D::T* col, int64_t ldw, int64_t k0, int64_t k1, F use)
    {
        int64_t k = k0;
        for (; k + (kColBatch - 1) * kDown < k1; k += kColBatch * kDown) {
            Piece q[kColBatch];
#pragma unroll
            for (int i = 0; i < kColBatch; ++i)
                q[i] = __ldg(reinterpret_cast<const Piece*>(col + (k + i * kDown) * ldw));
#pragma unroll
            for (int i = 0; i < kColBatch; ++i) use(k + i * kDown, q[i]);
        }
        for (; k < k1; k += kDown) use(k, __ldg(reinterpret_cast<const Piece*>(col + k * ldw)));
    }
};

template <class D, bool kVector, int kAcross>
__global__ void __launch_bounds__(kColThreads, kColBlocks)
int8_quantize_cols_kernel(const typename D::T* __restrict__ w, int64_t ldw, int8_t* __restrict__ codes,
                          int64_t ld_codes, float* __restrict__ scales, int64_t K, int64_t N)
{
    using S = Cols<D, kVector, kAcross>;
    constexpr int V = S::V;
    constexpr bool kPacked = V == 8;  // two 16-bit magnitudes compared at once
    constexpr int kMax = kPacked ? 4 : V;
    __shared__ uint32_t smax[S::kStrip];
    __shared__ float sinv[S::kStrip];
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, tx = tid % kAcross, ty = tid / kAcross;
    const int64_t e = blockIdx.y;
    const int64_t n0 = (int64_t)(blockIdx.x / ctas) * S::kStrip, n = n0 + tx * V;
    const int64_t share = (K + ctas - 1) / ctas;
    const int64_t k0 = min(K, rank * share), k1 = min(K, k0 + share);
    const typename D::T* src = w + e * K * ldw + n;
    const bool have = n < N;  // the vector form has N a multiple of V
    for (int i = tid; i < S::kStrip; i += kColThreads) smax[i] = 0u;
    __syncthreads();
    uint32_t m[kMax];
#pragma unroll
    for (int j = 0; j < kMax; ++j) m[j] = 0u;
    if (have)
        S::each(src, ldw, k0 + ty, k1, [&](int64_t, const typename S::Piece& q) {
            if constexpr (kPacked) {
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = __vmaxu2(m[j], u[j] & 0x7FFF7FFFu);
            } else if constexpr (kVector) {
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = max(m[j], u[j] & 0x7FFFFFFFu);
            } else {
                m[0] = max(m[0], magnitude(D::widen(q)));
            }
        });
#pragma unroll
    for (int j = 0; j < kMax; ++j) {
        if constexpr (kPacked) {  // widened, magnitudes still order as integers
            atomicMax(&smax[tx * V + 2 * j], magnitude(D::widen((uint16_t)m[j])));  // a maximum has no order
            atomicMax(&smax[tx * V + 2 * j + 1], magnitude(D::widen((uint16_t)(m[j] >> 16))));
        } else {
            atomicMax(&smax[tx * V + j], m[j]);
        }
    }
    cluster.sync();
    for (int i = tid; i < S::kStrip; i += kColThreads) {
        uint32_t a = 0u;
        for (int r = 0; r < ctas; ++r) a = max(a, *cluster.map_shared_rank(&smax[i], r));
        const RowScale rs = row_scale(a);
        sinv[i] = rs.inv;
        if (rank == 0 && n0 + i < N) scales[e * N + n0 + i] = rs.scale;
    }
    cluster.sync();  // also: no block leaves while another reads its smax
    if (!have) return;
    float inv[V];
    bool finite = true;  // all of this thread's columns
#pragma unroll
    for (int j = 0; j < V; ++j) {
        inv[j] = sinv[tx * V + j];
        finite = finite && inv[j] != 0.0f;
    }
    int8_t* dst = codes + e * K * ld_codes + n;
    const auto make = [&](auto all_finite) {
        S::each(src, ldw, k0 + ty, k1, [&](int64_t k, const typename S::Piece& q) {
            float v[V];
            if constexpr (kVector) D::widen(q, v);
            else v[0] = D::widen(q);
            uint32_t c[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                c[j] = code_bits(v[j], inv[j]);
                if (!decltype(all_finite)::value && inv[j] == 0.0f) c[j] = 0u;
            }
            int8_t* out = dst + k * ld_codes;
            if constexpr (kVector) {
                uint32_t u[V / 4];
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    u[j / 4] = __byte_perm(__byte_perm(c[j], c[j + 1], 0x0040),
                                           __byte_perm(c[j + 2], c[j + 3], 0x0040), 0x5410);
                if constexpr (V == 8) *reinterpret_cast<uint2*>(out) = make_uint2(u[0], u[1]);
                else *reinterpret_cast<uint32_t*>(out) = u[0];
            } else {
                *out = (int8_t)c[0];
            }
        });
    };
    if (finite) make(std::true_type());
    else make(std::false_type());
}

bool aligned(const void* p, int64_t ld_bytes, int to)
{
    return reinterpret_cast<uintptr_t>(p) % to == 0 && ld_bytes % to == 0;
}

template <class D>
cudaError_t rows(const void* x, int64_t ldx, int8_t* codes, int64_t ld_codes, float* scales, int64_t M, int64_t K,
                 cudaStream_t stream)
{
    const auto* in = static_cast<const typename D::T*>(x);
    const int words_ok = aligned(codes, ld_codes, D::kVec);
    const bool vec = words_ok && aligned(x, ldx * (int64_t)sizeof(typename D::T), 16);
    // A warp per row where rows are many and a warp can hold one; else a block per row.
    const bool warps = M >= 4 * (int64_t)device_sm_count() && (!vec || K <= (int64_t)32 * kHold * D::kVec);
    const int64_t per_block = warps ? kRowThreads / 32 : 1;
    const unsigned grid = (unsigned)std::min<int64_t>((M + per_block - 1) / per_block, (int64_t)device_sm_count() * 16);
    const auto kernel = vec ? (warps ? int8_quantize_rows_kernel<D, 32> : int8_quantize_rows_kernel<D, kRowThreads>)
                            : (warps ? int8_quantize_shifted_rows_kernel<D, 32>
                                     : int8_quantize_shifted_rows_kernel<D, kRowThreads>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = stream_captures(stream) ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, in, ldx, codes, ld_codes, scales, M, K, words_ok);
}

template <class D>
cudaError_t cols(const void* w, int64_t ldw, int8_t* codes, int64_t ld_codes, float* scales, int64_t E, int64_t K,
                 int64_t N, cudaStream_t stream)
{
    const auto* in = static_cast<const typename D::T*>(w);
    const bool vec = N % D::kVec == 0 && aligned(w, ldw * (int64_t)sizeof(typename D::T), 16) &&
                     aligned(codes, ld_codes, D::kVec);
    const int64_t sms = device_sm_count(), resident = kColBlocks * sms;
    int64_t strip = kColWide * (vec ? D::kVec : 1);
    // Blocks per strip: one for kColShare rows, more while SMs are without one (16 x 1024 x 4096
    // BF16: 46 us with 2, 62 with 8; 32 x 256 x 2048: 15 with 1, 53 with 8; 1 x 1024 x 4096: 6.8 with
    // 8, 9.1 with 2), fewer where they would only begin a second round (8192 x 8192: 57 us with 4
    // in one round, 61 with 8 in 1.15).
    const auto blocks = [&](int64_t ctas) { return (N + strip - 1) / strip * E * ctas; };
    int ctas = 1;
    while (ctas < kColCtas && (K > kColShare * ctas || blocks(ctas) < sms)) ctas *= 2;
    if (ctas > 1 && blocks(ctas) > resident && blocks(ctas) * 4 <= resident * 5) ctas /= 2;
    // Strips half as wide where SMs are still without a block (4001 x 1000 FP16: 12.5 -> 11.1 us).
    const bool narrow = vec && blocks(ctas) < sms;
    if (narrow) strip /= 2;
    const auto kernel = narrow ? int8_quantize_cols_kernel<D, true, kColWide / 2>
                        : vec  ? int8_quantize_cols_kernel<D, true, kColWide>
                               : int8_quantize_cols_kernel<D, false, kColWide>;
    constexpr int64_t kMaxGridY = 65535;
    for (int64_t e = 0; e < E; e += kMaxGridY) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((N + strip - 1) / strip) * ctas, (unsigned)std::min(kMaxGridY, E - e));
        cfg.blockDim = dim3(kColThreads);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, in + e * K * ldw, ldw, codes + e * K * ld_codes,
                                                   ld_codes, scales + e * N, K, N);
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_int8_quantize_rows(const void* x, int type, int64_t ldx, int8_t* codes, int64_t ld_codes,
                                      float* scales, int64_t M, int64_t K, cudaStream_t stream)
{
    if (M == 0) return cudaSuccess;
    if (type == MPK_TYPE_F32) return rows<F32>(x, ldx, codes, ld_codes, scales, M, K, stream);
    if (type == MPK_TYPE_BF16) return rows<Bf16>(x, ldx, codes, ld_codes, scales, M, K, stream);
    return rows<F16>(x, ldx, codes, ld_codes, scales, M, K, stream);
}

cudaError_t launch_int8_quantize_cols(const void* w, int type, int64_t ldw, int8_t* codes, int64_t ld_codes,
                                      float* scales, int64_t E, int64_t K, int64_t N, cudaStream_t stream)
{
    if (E == 0 || N == 0) return cudaSuccess;
    if (type == MPK_TYPE_F32) return cols<F32>(w, ldw, codes, ld_codes, scales, E, K, N, stream);
    if (type == MPK_TYPE_BF16) return cols<Bf16>(w, ldw, codes, ld_codes, scales, E, K, N, stream);
    return cols<F16>(w, ldw, codes, ld_codes, scales, E, K, N, stream);
}

}  // namespace mpk
