// Quantizers to 8-bit integers with one FP32 scale per row (token) or per column
// (output channel of a weight).  HBM bound.
// The numerics are int8_codes.cuh's.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "int8_codes.cuh"
#include "mpk.h"
#include "mpk_internal.h"
#include "mpk_ptx.cuh"

namespace mpk {
namespace {

namespace cg = cooperative_groups;

using namespace int8;

// ------------------------------- rows ---------------------------------------
// One block per row (the grid strides over the rows): a pass for the largest
// magnitude, a pass for the codes, which finds the row in L1 or L2.
constexpr int kRowThreads = 256;

template <class D, bool kVector>
__global__ void __launch_bounds__(kRowThreads)
int8_quantize_rows_kernel(const typename D::T* __restrict__ x, int64_t ldx, int8_t* __restrict__ codes,
                          int64_t ld_codes, float* __restrict__ scales, int64_t M, int64_t K)
{
    allow_dependent_launch();
    __shared__ uint32_t warp_max[kRowThreads / 32];
    const int tid = threadIdx.x;
    const int64_t nvec = kVector ? K / D::kVec : 0;
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const typename D::T* row = x + m * ldx;
        int8_t* out = codes + m * ld_codes;
        uint32_t amax = 0;
        for (int64_t i = tid; i < nvec; i += kRowThreads) {
            float v[D::kVec];
            D::widen(__ldg(reinterpret_cast<const uint4*>(row) + i), v);
#pragma unroll
            for (int j = 0; j < D::kVec; ++j) amax = max(amax, magnitude(v[j]));
        }
        for (int64_t k = nvec * D::kVec + tid; k < K; k += kRowThreads) amax = max(amax, magnitude(D::widen(row[k])));
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        if ((tid & 31) == 0) warp_max[tid >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kRowThreads / 32; ++w) amax = max(amax, warp_max[w]);
        const RowScale rs = row_scale(amax);
        if (tid == 0) scales[m] = rs.scale;
        for (int64_t i = tid; i < nvec; i += kRowThreads) {
            float v[D::kVec];
            D::widen(__ldg(reinterpret_cast<const uint4*>(row) + i), v);
#pragma unroll
            for (int j = 0; j < D::kVec; j += 4)
                *reinterpret_cast<uint32_t*>(out + i * D::kVec + j) = pack4(v + j, rs.inv);
        }
        for (int64_t k = nvec * D::kVec + tid; k < K; k += kRowThreads)
            out[k] = rs.inv == 0.0f ? (int8_t)0 : (int8_t)code_bits(D::widen(row[k]), rs.inv);
        __syncthreads();  // warp_max is read before the next row writes it
    }
}

// ------------------------------ columns -------------------------------------
// A cluster of kColCtas blocks per strip of columns and expert: each block takes a
// share of the rows, the strip's largest magnitudes are joined through distributed
// shared memory, and a second pass over the share (found in L2) makes the codes.
constexpr int kColThreads = 256, kColCtas = 8;

template <class D, bool kVector>
__global__ void __launch_bounds__(kColThreads)
int8_quantize_cols_kernel(const typename D::T* __restrict__ w, int64_t ldw, int8_t* __restrict__ codes,
                          int64_t ld_codes, float* __restrict__ scales, int64_t K, int64_t N)
{
    constexpr int V = kVector ? D::kVec : 1;
    constexpr int kAcross = kVector ? 128 / D::kVec : 32;  // threads across the strip
    constexpr int kStrip = kAcross * V;
    constexpr int kDown = kColThreads / kAcross;           // rows per step
    __shared__ uint32_t smax[kStrip];
    __shared__ float sinv[kStrip];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x;
    const int tx = tid % kAcross, ty = tid / kAcross;
    const int64_t e = blockIdx.y;
    const int rank = blockIdx.x % kColCtas;
    const int64_t n0 = (int64_t)(blockIdx.x / kColCtas) * kStrip;
    const int64_t n = n0 + tx * V;
    const int64_t share = (K + kColCtas - 1) / kColCtas;
    const int64_t k0 = min(K, rank * share), k1 = min(K, k0 + share);
    const typename D::T* src = w + e * K * ldw;
    int8_t* dst = codes + e * K * ld_codes;
    for (int i = tid; i < kStrip; i += kColThreads) smax[i] = 0u;
    __syncthreads();
    uint32_t amax[V];
#pragma unroll
    for (int j = 0; j < V; ++j) amax[j] = 0u;
    if (n < N) {  // the vector form has N a multiple of V
        for (int64_t k = k0 + ty; k < k1; k += kDown) {
            float v[V];
            if constexpr (kVector) D::widen(__ldg(reinterpret_cast<const uint4*>(src + k * ldw + n)), v);
            else v[0] = D::widen(src[k * ldw + n]);
#pragma unroll
            for (int j = 0; j < V; ++j) amax[j] = max(amax[j], magnitude(v[j]));
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) atomicMax(&smax[tx * V + j], amax[j]);  // a maximum has no order
    cluster.sync();
    for (int i = tid; i < kStrip; i += kColThreads) {
        uint32_t a = 0u;
        for (int r = 0; r < kColCtas; ++r) a = max(a, *cluster.map_shared_rank(&smax[i], r));
        const RowScale rs = row_scale(a);
        sinv[i] = rs.inv;
        if (rank == 0 && n0 + i < N) scales[e * N + n0 + i] = rs.scale;
    }
    cluster.sync();  // also: no block leaves while another reads its smax
    if (n >= N) return;
    float inv[V];
#pragma unroll
    for (int j = 0; j < V; ++j) inv[j] = sinv[tx * V + j];
    for (int64_t k = k0 + ty; k < k1; k += kDown) {
        float v[V];
        if constexpr (kVector) D::widen(__ldg(reinterpret_cast<const uint4*>(src + k * ldw + n)), v);
        else v[0] = D::widen(src[k * ldw + n]);
        uint32_t b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) b[j] = inv[j] == 0.0f ? 0u : code_bits(v[j], inv[j]);
        int8_t* out = dst + k * ld_codes + n;
        if constexpr (kVector) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
                *reinterpret_cast<uint32_t*>(out + j) =
                    __byte_perm(__byte_perm(b[j], b[j + 1], 0x0040), __byte_perm(b[j + 2], b[j + 3], 0x0040), 0x5410);
        } else {
            *out = (int8_t)b[0];
        }
    }
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
    const unsigned grid = (unsigned)std::min<int64_t>(M, (int64_t)device_sm_count() * 8);
    if (aligned(x, ldx * (int64_t)sizeof(typename D::T), 16) && aligned(codes, ld_codes, 4))
        int8_quantize_rows_kernel<D, true><<<grid, kRowThreads, 0, stream>>>(in, ldx, codes, ld_codes, scales, M, K);
    else
        int8_quantize_rows_kernel<D, false><<<grid, kRowThreads, 0, stream>>>(in, ldx, codes, ld_codes, scales, M, K);
    return cudaGetLastError();
}

template <class D>
cudaError_t cols(const void* w, int64_t ldw, int8_t* codes, int64_t ld_codes, float* scales, int64_t E, int64_t K,
                 int64_t N, cudaStream_t stream)
{
    const auto* in = static_cast<const typename D::T*>(w);
    const bool vec = N % D::kVec == 0 && aligned(w, ldw * (int64_t)sizeof(typename D::T), 16) &&
                     aligned(codes, ld_codes, 4);
    const int64_t strip = vec ? 128 : 32;
    const auto kernel = vec ? int8_quantize_cols_kernel<D, true> : int8_quantize_cols_kernel<D, false>;
    constexpr int64_t kMaxGridY = 65535;
    for (int64_t e = 0; e < E; e += kMaxGridY) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((N + strip - 1) / strip) * kColCtas, (unsigned)std::min(kMaxGridY, E - e));
        cfg.blockDim = dim3(kColThreads);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = kColCtas;
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
