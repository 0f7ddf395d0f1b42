// Grouped products: host side of the tcgen05 kernel (gemm_grouped.cuh), the plain kernel for what bulk
// copies cannot address, and the C entry points b200_gemm_grouped and b200_gemm_grouped_k.
#include "gemm_grouped.cuh"

#include <algorithm>
#include <atomic>

#include "internal.h"
#include "tensor_map.h"

namespace b200 {
namespace {

// ---------------------------------------------------------------------------------------------
// plain kernel: 64 x 64 tiles, binary32 FMA, any leading dimension and alignment
// ---------------------------------------------------------------------------------------------
constexpr int kTile = 64, kTileK = 16;

__device__ __forceinline__ float widen16(unsigned short raw, int bf16) {
    return bf16 ? __uint_as_float(static_cast<uint32_t>(raw) << 16) : __half2float(__ushort_as_half(raw));
}
__device__ __forceinline__ float load_as_float(const void* p, long long i, int fmt) {
    return fmt == 0 ? static_cast<const float*>(p)[i] : widen16(static_cast<const unsigned short*>(p)[i], fmt == 2);
}
__device__ __forceinline__ void store_from_float(void* p, long long i, int fmt, float v) {
    if (fmt == 0) static_cast<float*>(p)[i] = v;
    else if (fmt == 1) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

struct PlainTile {
    const unsigned short* A;  // element (m, k) at m * am + k * ak
    long long am, ak;
    const unsigned short* B;  // element (k, n) at k * bk + n * bn
    long long bk, bn;
    long long m0, n0, M, N, K0, K1;  // rows < M, columns < N, k in [K0, K1)
};

// One 64 x 64 tile; 256 threads; kAk: A is contiguous along k (threads of a warp walk along k then).
template <bool kAk, bool kBk>
__device__ __forceinline__ void plain_tile(const PlainTile& t, int ab_bf16, float (&acc)[4][4], float (*sA)[kTile + 1], float (*sB)[kTile + 1]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (long long k0 = t.K0; k0 < t.K1; k0 += kTileK) {
        for (int e = threadIdx.x; e < kTile * kTileK; e += 256) {
            const int mm = kAk ? e / kTileK : e % kTile, ka = kAk ? e % kTileK : e / kTile;
            const int nn = kBk ? e / kTileK : e % kTile, kb = kBk ? e % kTileK : e / kTile;
            sA[ka][mm] = (t.m0 + mm < t.M && k0 + ka < t.K1) ? widen16(t.A[(t.m0 + mm) * t.am + (k0 + ka) * t.ak], ab_bf16) : 0.f;
            sB[kb][nn] = (t.n0 + nn < t.N && k0 + kb < t.K1) ? widen16(t.B[(k0 + kb) * t.bk + (t.n0 + nn) * t.bn], ab_bf16) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kTileK; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sA[kk][tx * 4 + i], sB[kk][ty * 4 + j], acc[i][j]);
        __syncthreads();
    }
}

struct PlainParams {
    const unsigned short *A, *B;
    long long lda, ldb, stride_a;
    const void* C;
    void* D;
    long long ldc, ldd, stride_c, stride_d;
    long long M, N, K;
    int groups, ab_bf16, c_fmt, d_fmt;
    float alpha, beta;
    const int* offsets;
    int* status;
};

__device__ __forceinline__ void plain_store(const PlainParams& p, const float (&acc)[4][4], long long m0, long long n0, long long n_end, int e,
                                            bool per_group) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int j = 0; j < 4; ++j)
        for (int i = 0; i < 4; ++i) {
            const long long m = m0 + tx * 4 + i, n = n0 + ty * 4 + j;
            if (m >= p.M || n >= n_end) continue;
            float v = p.alpha * acc[i][j];
            if (p.beta != 0.0f) v = fmaf(p.beta, load_as_float(p.C, m + n * p.ldc + (per_group ? e * p.stride_c : 0), p.c_fmt), v);
            store_from_float(p.D, m + n * p.ldd + (per_group ? e * p.stride_d : 0), p.d_fmt, v);
        }
}

template <bool kTransA>
__global__ void __launch_bounds__(256) grouped_plain_kernel(const PlainParams p) {
    __shared__ float sA[kTileK][kTile + 1], sB[kTileK][kTile + 1];
    __shared__ int off[kMaxGroups + 1], first[kMaxGroups + 1];
    __shared__ unsigned long long sums[8];
    if (!load_groups<true>(p.offsets, p.groups, static_cast<int>(p.N), kTile, off, first, sums)) {
        if (threadIdx.x == 0) report_bad_offsets(p.status, p.groups);
        return;
    }
    for (int q = blockIdx.y; q < first[p.groups]; q += gridDim.y) {
        const int e = find_group(first, p.groups, q);
        const long long m0 = static_cast<long long>(blockIdx.x) * kTile, n0 = off[e] + static_cast<long long>(q - first[e]) * kTile;
        float acc[4][4] = {};
        const PlainTile t = {p.A + e * p.stride_a, kTransA ? p.lda : 1, kTransA ? 1 : p.lda, p.B, 1, p.ldb, m0, n0, p.M, off[e + 1], 0, p.K};
        plain_tile<kTransA, true>(t, p.ab_bf16, acc, sA, sB);
        plain_store(p, acc, m0, n0, off[e + 1], e, false);
    }
}

__global__ void __launch_bounds__(256) grouped_k_plain_kernel(const PlainParams p) {
    __shared__ float sA[kTileK][kTile + 1], sB[kTileK][kTile + 1];
    __shared__ int off[kMaxGroups + 1];
    if (!load_groups<false>(p.offsets, p.groups, static_cast<int>(p.K), kTile, off, nullptr, nullptr)) {
        if (threadIdx.x == 0) report_bad_offsets(p.status, p.groups);
        return;
    }
    const long long m0 = static_cast<long long>(blockIdx.x) * kTile, n0 = static_cast<long long>(blockIdx.y) * kTile;
    for (int e = blockIdx.z; e < p.groups; e += gridDim.z) {
        float acc[4][4] = {};
        const PlainTile t = {p.A, 1, p.lda, p.B, p.ldb, 1, m0, n0, p.M, p.N, off[e], off[e + 1]};
        plain_tile<false, false>(t, p.ab_bf16, acc, sA, sB);
        plain_store(p, acc, m0, n0, p.N, e, true);
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
struct Grouped {
    bool ragged_k;
    int transA;
    int64_t M, N, K, groups;
    float alpha, beta;
    const void *A, *B, *C;
    void* D;
    int64_t lda, stride_a, ldb, ldc, stride_c, ldd, stride_d;
    int ab_type, c_type, d_type;
    const int32_t* offsets;
};

template <int kBN, bool kAMn, bool kRaggedK, int kCtas, int kSums, int kSplit>
int launch_sums(const CUtensorMap (&tm)[2], const GroupedParams& p, int grid, cudaStream_t stream, bool pdl) {
    using Cfg = GroupedCfg<kBN, kRaggedK, kCtas, kSums, kSplit>;
    auto kern = gemm_grouped_tcgen05<kBN, kAMn, kRaggedK, kCtas, kSums, kSplit>;
    static std::atomic<uint64_t> done{0};  // devices that have been opted in to the kernel's shared memory
    int dev = 0;
    B200_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !((done.load(std::memory_order_relaxed) >> dev) & 1u)) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
        // the kernel deals out 168 registers a thread among its warpgroups: one built with fewer would wait for more
        cudaFuncAttributes at;
        B200_CUDA_TRY(cudaFuncGetAttributes(&at, kern));
        if (at.numRegs != 168) return fail(B200_UNSUPPORTED, "grouped gemm: kernel built with " + std::to_string(at.numRegs) + " registers, not 168");
        if (dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kSplit > 1 ? kSplit : kCtas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm[0], tm[1], p));
    return B200_OK;
}

// binary32 results, and long sums of 16-bit ones, add several accumulators with rounding to nearest (epilogue_sm100.cuh)
template <int kBN, bool kAMn, bool kRaggedK, int kCtas>
int launch_grouped(const CUtensorMap (&tm)[2], const GroupedParams& p, int grid, cudaStream_t stream, bool pdl) {
    constexpr int kSplit = kBN == 32 ? 2 : 1;  // few columns per group: pairs of CTAs that may share a tile's inner dimension
    if (p.e.d_fmt == 0) return launch_sums<kBN, kAMn, kRaggedK, kCtas, kBinary32, kSplit>(tm, p, grid, stream, pdl);
    if (p.K > p.e.whole_kb * 64) return launch_sums<kBN, kAMn, kRaggedK, kCtas, kLongSums, kSplit>(tm, p, grid, stream, pdl);
    return launch_sums<kBN, kAMn, kRaggedK, kCtas, kOneAccumulator, kSplit>(tm, p, grid, stream, pdl);
}

template <int kBN, int kCtas>
int launch_kind(const Grouped& g, const CUtensorMap (&tm)[2], const GroupedParams& p, int grid, cudaStream_t stream, bool pdl) {
    if (g.ragged_k) {
        if constexpr ((kBN / kCtas) % 64 == 0) return launch_grouped<kBN, true, true, kCtas>(tm, p, grid, stream, pdl);
        else return fail(B200_UNSUPPORTED, "grouped_k: 64 tile columns per CTA at least");
    }
    if (g.transA) return launch_grouped<kBN, false, false, kCtas>(tm, p, grid, stream, pdl);
    return launch_grouped<kBN, true, false, kCtas>(tm, p, grid, stream, pdl);
}

bool eligible(const Grouped& g, std::string* why) {
    auto no = [&](const char* m) {
        *why = m;
        return false;
    };
    if (g.K <= 0) return no("K is 0");
    if ((reinterpret_cast<uintptr_t>(g.A) | reinterpret_cast<uintptr_t>(g.B)) & 15u) return no("A and B must be 16-byte aligned for TMA");
    if (g.lda % 8 || g.ldb % 8) return no("lda and ldb must be multiples of 8 elements for TMA");
    if (!g.ragged_k && g.groups > 1 && g.stride_a != 0) {
        if (g.stride_a % 8) return no("stride_a must be a multiple of 8 elements for TMA");
        if (g.stride_a < g.lda * (g.transA ? g.M : g.K)) return no("stride_a must be at least the extent of one matrix");
    }
    return true;
}

// How many clusters of four CTAs the current device holds at once: fewer than SMs / 4, since a cluster lies within one
// part of the chip and those have no multiple of four SMs (33 of 37 on a B200).
int resident_clusters(int* clusters) {
    static std::atomic<int> known[64];  // per device
    int dev = 0;
    B200_CUDA_TRY(cudaGetDevice(&dev));
    *clusters = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (*clusters > 0) return B200_OK;
    auto kern = gemm_grouped_tcgen05<64, true, true, 1, kBinary32, 4>;
    using Cfg = GroupedCfg<64, true, 1, kBinary32, 4>;
    B200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 4;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(4, 1, 1);
    cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    B200_CUDA_TRY(cudaOccupancyMaxActiveClusters(clusters, kern, &cfg));
    if (dev < 64) known[dev].store(*clusters, std::memory_order_relaxed);
    return B200_OK;
}

// Few tiles and a long inner dimension: clusters of four CTAs share each tile's K (64-column tiles), in as many rounds as
// the clusters that the device holds need.  Measured, whole tiles against shared ones, the last number of tiles of each
// round: one round K = 1024 9.3 / 11.5 us, K = 1536 11.8 / 12.1 (16 tiles 11.8 / 10.5), K = 2048 14.2 / 12.6; two rounds K = 3000 19.0 / 19.1, K =
// 4096 23.8 / 20.1; three K = 4096 23.9 / 26.2, K = 6000 34.2 / 33.6, K = 8192 46.3 / 42.7; four K = 16384 87.8 / 90.0.
// Ragged K: by the mean length; a longer group than the others takes more from whole tiles than from shared ones.
bool may_share_k(const b200_handle* h, const Grouped& g) {
    if (h->tile_n != 0 || h->cta_pair != 0 || h->max_ctas != 0) return false;
    if (!g.ragged_k && g.N <= 32 * g.groups) return false;  // 32-column tiles, in pairs
    return (g.ragged_k ? g.K / g.groups : g.K) >= 1536;
}
bool shares_k(const Grouped& g, int clusters) {
    const int64_t cols = g.ragged_k ? g.groups * ((g.N + 63) / 64) : g.N / 64 + std::min(g.groups, g.N);
    const int64_t units = cols * ((g.M + 127) / 128), k = g.ragged_k ? g.K / g.groups : g.K;
    const int64_t rounds = (units + clusters - 1) / std::max(clusters, 1);
    return clusters > 0 && rounds <= 3 && k >= (rounds == 1 ? 1536 : int64_t(2048) << (rounds - 1));
}

// Tile columns.  Ragged N: the sizes of the groups are not known here, their mean is.  Wide tiles read
// each A_e less often; the instruction's N follows the columns that a group really has.
void pick_tile(const b200_handle* h, const Grouped& g, int* tile_n, int* pair) {
    *tile_n = h->tile_n;
    if (*tile_n == 0) {
        const int64_t n = g.ragged_k ? g.N : (g.N + g.groups - 1) / g.groups;
        *tile_n = n > 128 ? 256 : n > 64 ? 128 : (n > 32 || g.ragged_k) ? 64 : 32;
    }
    *pair = h->cta_pair;
    if (*pair == 0) *pair = (*tile_n == 256 && g.M > 128) ? 2 : 1;
    if (*pair == 2 && *tile_n < 128) *pair = 1;
    if (*pair == 1 && *tile_n == 256) *tile_n = 128;
}

int run_tcgen05(b200_handle* h, cudaStream_t stream, const Grouped& g) {
    int tile_n, pair, rc;
    pick_tile(h, g, &tile_n, &pair);
    bool share = may_share_k(h, g);
    int clusters = 0;
    if (share) {
        if ((rc = resident_clusters(&clusters))) return rc;
        share = shares_k(g, clusters);
    }
    if (share) {
        tile_n = 64;
        pair = 1;
    }
    GroupedParams p = {};
    p.e.M = static_cast<int>(g.M);
    p.N = static_cast<int>(g.N);
    p.K = static_cast<int>(g.K);
    p.groups = static_cast<int>(g.groups);
    const int64_t tiles_m = (g.M + 128 * pair - 1) / (128 * pair), tiles_n = (g.N + tile_n - 1) / tile_n;
    p.e.alpha = g.alpha;
    p.e.beta = g.beta;
    p.offsets = g.offsets;
    p.e.C = g.C;
    p.e.D = g.D;
    p.e.ldc = g.ldc;
    p.e.ldd = g.ldd;
    p.e.stride_c = g.stride_c;
    p.e.stride_d = g.stride_d;
    p.e.c_fmt = elem_fmt(g.c_type);
    p.e.d_fmt = elem_fmt(g.d_type);
    p.e.whole_kb = whole_kb(p.e.d_fmt);
    p.a_per_group = g.stride_a != 0 ? 1 : 0;
    p.ab_bf16 = g.ab_type == B200_BF16 ? 1 : 0;
    p.status = h->status_word;
    p.wait_budget_ns = h->wait_budget_ns;

    const int bn_local = tile_n / pair, bbox = std::min(bn_local, 64);
    const CUtensorMapDataType dt = map_type(g.ab_type);
    CUtensorMap tm[2];
    if (g.ragged_k) {
        if ((rc = encode_map_2d(&tm[0], dt, 2, g.A, g.M, g.K, g.lda, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B, "A"))) return rc;
        if ((rc = encode_map_2d(&tm[1], dt, 2, g.B, g.N, g.K, g.ldb, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B, "B"))) return rc;
    } else {
        BatchDim b;
        b.count = g.stride_a != 0 ? g.groups : 1;
        b.stride = b.count > 1 ? g.stride_a : g.lda * (g.transA ? g.M : g.K);
        if (g.transA) rc = encode_map_2d(&tm[0], dt, 2, g.A, g.K, g.M, g.lda, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B, "A (row-major)", b);
        else rc = encode_map_2d(&tm[0], dt, 2, g.A, g.M, g.K, g.lda, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B, "A (column-major)", b);
        if (rc) return rc;
        if ((rc = encode_map_2d(&tm[1], dt, 2, g.B, g.K, g.N, g.ldb, 64, bbox, CU_TENSOR_MAP_SWIZZLE_128B, "B"))) return rc;
    }
    p.e.d_pairs = !(reinterpret_cast<uintptr_t>(g.D) & 3u) && g.ldd % 2 == 0 && g.stride_d % 2 == 0;

    // ragged N: at most one partial tile column per group that has columns
    const int64_t cols = g.ragged_k ? g.groups * tiles_n : g.N / tile_n + std::min<int64_t>(g.groups, g.N);
    const int64_t units = cols * tiles_m;
    if (units > 0x7fffff00ll) return fail(B200_UNSUPPORTED, "grouped gemm: too many tiles for one launch");
    p.raster = Raster::of(h->raster_group > 0 ? h->raster_group : 8, static_cast<int>(tiles_m));
    if (g.ragged_k) {
        p.tiles_n = static_cast<int>(tiles_n);
        p.tiles = Divisor::of(static_cast<int>(tiles_m * tiles_n));
    }
    int cap = h->max_ctas > 0 ? std::min(h->max_ctas, h->sm_count) : h->sm_count;
    int grid = static_cast<int>(std::min<int64_t>(std::max(cap / pair, 1), units)) * pair;
    if (tile_n == 32) grid = std::max(cap / 2, 1) * 2;  // pairs of CTAs; how many tiles there are is not known here
    const bool pdl = h->pdl != 0;
    if (share) {
        grid = static_cast<int>(std::min<int64_t>(clusters, units)) * 4;
        if (g.ragged_k) rc = launch_sums<64, true, true, 1, kBinary32, 4>(tm, p, grid, stream, pdl);
        else if (g.transA) rc = launch_sums<64, false, false, 1, kBinary32, 4>(tm, p, grid, stream, pdl);
        else rc = launch_sums<64, true, false, 1, kBinary32, 4>(tm, p, grid, stream, pdl);
    } else if (pair == 2) rc = tile_n == 256 ? launch_kind<256, 2>(g, tm, p, grid, stream, pdl) : launch_kind<128, 2>(g, tm, p, grid, stream, pdl);
    else if (tile_n == 128) rc = launch_kind<128, 1>(g, tm, p, grid, stream, pdl);
    else if (tile_n == 64) rc = launch_kind<64, 1>(g, tm, p, grid, stream, pdl);
    else rc = launch_kind<32, 1>(g, tm, p, grid, stream, pdl);
    if (rc) return rc;
    h->last = {B200_KERNEL_TCGEN05, tile_n, share ? 4 : 1, grid, pair};
    return B200_OK;
}

int run_plain(b200_handle* h, cudaStream_t stream, const Grouped& g) {
    PlainParams p = {static_cast<const unsigned short*>(g.A), static_cast<const unsigned short*>(g.B), g.lda, g.ldb, g.stride_a, g.C, g.D,
                     g.ldc, g.ldd, g.stride_c, g.stride_d, g.M, g.N, g.K, static_cast<int>(g.groups), g.ab_type == B200_BF16 ? 1 : 0,
                     elem_fmt(g.c_type), elem_fmt(g.d_type), g.alpha, g.beta, g.offsets, h->status_word};
    const int64_t gx = (g.M + kTile - 1) / kTile;
    const int64_t gy = g.ragged_k ? (g.N + kTile - 1) / kTile : std::min<int64_t>(g.N / kTile + std::min(g.groups, g.N), 65535);
    if (gy > 65535) return fail(B200_UNSUPPORTED, "grouped gemm: N too large for one launch of the simple kernel");
    dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy), g.ragged_k ? static_cast<unsigned>(g.groups) : 1u);
    if (g.ragged_k) grouped_k_plain_kernel<<<grid, 256, 0, stream>>>(p);
    else if (g.transA) grouped_plain_kernel<true><<<grid, 256, 0, stream>>>(p);
    else grouped_plain_kernel<false><<<grid, 256, 0, stream>>>(p);
    B200_CUDA_TRY(cudaGetLastError());
    h->last = {B200_KERNEL_SIMPLE, kTile, 1, static_cast<int>(grid.x * grid.y * grid.z), 1};
    return B200_OK;
}

bool is_elem_type(int t) { return t == B200_F16 || t == B200_F32 || t == B200_BF16; }

int check(const Grouped& g) {
    const std::string name = g.ragged_k ? "grouped_k: " : "grouped: ";
    auto bad = [&](const char* m) { return fail(B200_INVALID_ARG, name + m); };
    const int64_t most = 0x7fffff00ll;
    if (g.ab_type != B200_F16 && g.ab_type != B200_BF16) return bad("invalid element type: A and B must be Float16 or bfloat16");
    if (!is_elem_type(g.c_type) || !is_elem_type(g.d_type)) return bad("invalid element type: C and D must be Float16, bfloat16 or Float32");
    if (g.M < 0 || g.N < 0 || g.K < 0) return bad("negative dimension");
    if (g.M > most || g.N > most || g.K > most) return bad("dimension exceeds 2^31");
    if (g.groups < 0 || g.groups > kMaxGroups) return bad("groups must be in [0, 1024]");
    if (g.transA != 0 && g.transA != 1) return bad("transA must be 0 or 1");
    if (g.lda < std::max<int64_t>(1, g.transA ? g.K : g.M)) return bad("lda smaller than the rows of stored A");
    if (g.ldb < std::max<int64_t>(1, g.ragged_k ? g.N : g.K)) return bad("ldb smaller than the rows of stored B");
    if (g.ldd < std::max<int64_t>(1, g.M)) return bad("ldd smaller than M");
    if (g.beta != 0.0f && g.ldc < std::max<int64_t>(1, g.M)) return bad("ldc smaller than M");
    if (g.stride_a < 0 || g.stride_c < 0 || g.stride_d < 0) return bad("negative stride");
    if (g.ragged_k && g.groups > 1 && g.stride_d < g.ldd * g.N) return bad("stride_d smaller than one D matrix (results would overlap)");
    if (g.M == 0 || g.N == 0 || g.groups == 0) return B200_OK;
    if (!g.offsets) return bad("offsets is null");
    if (!g.D) return bad("D is null");
    if (g.beta != 0.0f && !g.C) return bad("C is null but beta != 0");
    if (g.K > 0 && (!g.A || !g.B)) return bad("A or B is null");
    const uintptr_t a = reinterpret_cast<uintptr_t>(g.A) | reinterpret_cast<uintptr_t>(g.B);
    if (reinterpret_cast<uintptr_t>(g.offsets) % 4 || a % 2 || reinterpret_cast<uintptr_t>(g.D) % elem_bytes(g.d_type) ||
        (g.beta != 0.0f && reinterpret_cast<uintptr_t>(g.C) % elem_bytes(g.c_type)))
        return bad("a pointer is not aligned to its element type");
    return B200_OK;
}

int entry(b200_handle* h, cudaStream_t stream, const Grouped& g) {
    int rc = check(g);
    if (rc) return rc;
    if (g.M == 0 || g.N == 0 || g.groups == 0) return B200_OK;
    if ((rc = poll_previous_launch(h)) || (rc = check_current_device(h))) return rc;
    std::string why;
    const bool ok = eligible(g, &why);
    if (h->force_kernel == B200_KERNEL_TCGEN05 && !ok) return fail(B200_UNSUPPORTED, "tcgen05 kernel not eligible: " + why);
    rc = (ok && h->force_kernel != B200_KERNEL_SIMPLE) ? run_tcgen05(h, stream, g) : run_plain(h, stream, g);
    return rc ? rc : note_launch(h, stream);
}

}  // namespace
}  // namespace b200

extern "C" int b200_gemm_grouped(b200_handle* h, b200_stream stream, int transA, int64_t M, int64_t N, int64_t K, float alpha,
                                 const void* A, int64_t lda, int64_t stride_a, const void* B, int64_t ldb, int ab_type, float beta,
                                 const void* C, int64_t ldc, int c_type, void* D, int64_t ldd, int d_type, const int32_t* offsets,
                                 int64_t groups) {
    if (!h) return b200::fail(B200_INVALID_ARG, "null handle");
    const b200::Grouped g = {false, transA, M, N, K, groups, alpha, beta, A, B, C, D, lda, stride_a, ldb, ldc, 0, ldd, 0, ab_type, c_type, d_type, offsets};
    return b200::entry(h, static_cast<cudaStream_t>(stream), g);
}

extern "C" int b200_gemm_grouped_k(b200_handle* h, b200_stream stream, int64_t M, int64_t N, int64_t K, float alpha, const void* A,
                                   int64_t lda, const void* B, int64_t ldb, int ab_type, float beta, const void* C, int64_t ldc,
                                   int64_t stride_c, int c_type, void* D, int64_t ldd, int64_t stride_d, int d_type,
                                   const int32_t* offsets, int64_t groups) {
    if (!h) return b200::fail(B200_INVALID_ARG, "null handle");
    const b200::Grouped g = {true, 0, M, N, K, groups, alpha, beta, A, B, C, D, lda, 0, ldb, ldc, stride_c, ldd, stride_d, ab_type, c_type, d_type, offsets};
    return b200::entry(h, static_cast<cudaStream_t>(stream), g);
}
