// Host side of the microscaled 4-bit products: b200_gemm_mxfp4 and b200_gemm_mxfp4_grouped.
#include "gemm_mxfp4.cuh"

#include <algorithm>
#include <atomic>

#include "internal.h"
#include "tensor_map.h"

namespace b200 {
namespace {

struct MxProblem {
    int64_t M, N, K, groups;
    float alpha, beta;
    const void *A, *SA, *B, *SB, *C;
    void* D;
    int64_t lda, stride_a, ldb, ldc, ldd;
    int c_type, d_type;
    const int32_t* offsets;
};

template <int kBN, int kCtas, bool kLong>
int launch_as(const CUtensorMap (&tm)[4], const MxGemmParams& p, int grid, cudaStream_t stream, bool pdl) {
    constexpr bool kSplit = kBN == 32;  // few columns: pairs of CTAs that may share a tile's inner dimension
    using Cfg = MxCfg<kBN, kCtas, kSplit>;
    auto kern = gemm_mxfp4_tcgen05<kBN, kCtas, kSplit, kLong>;
    static std::atomic<uint64_t> done{0};  // devices that have been opted in to the kernel's shared memory
    int dev = 0;
    B200_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !((done.load(std::memory_order_relaxed) >> dev) & 1u)) {
        B200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
        // the kernel deals out 128 registers a thread among its warpgroups: one built with fewer would wait for more
        cudaFuncAttributes at;
        B200_CUDA_TRY(cudaFuncGetAttributes(&at, kern));
        if (at.numRegs != 128) return fail(B200_UNSUPPORTED, "mxfp4 gemm: kernel built with " + std::to_string(at.numRegs) + " registers, not 128");
        if (dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kSplit ? 2 : kCtas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm[0], tm[1], tm[2], tm[3], p));
    return B200_OK;
}

template <int kBN, int kCtas>
int launch(const CUtensorMap (&tm)[4], const MxGemmParams& p, int grid, cudaStream_t stream, bool pdl) {
    if (p.K > p.e.whole_kb * 256) return launch_as<kBN, kCtas, true>(tm, p, grid, stream, pdl);  // more than one accumulator sums
    return launch_as<kBN, kCtas, false>(tm, p, grid, stream, pdl);
}

// Tile columns, by the mean length of the groups.  256 columns leave tensor memory for one accumulator: its
// reading out is not hidden, nor is C read ahead.  192 have two.  Measured in turn, 256 against 192: 8192 x 8192, K =
// 8192 210 / 250 us, K = 512 50 / 48 us; with a Float32 C, 8192 x 8192, K = 1024 118 / 111 us, K = 4096 149 / 160 us,
// and where two rounds of tiles are all there is, 4100 x 1111, K = 4096 33 / 24 us.
void pick_tile(const b200_handle* h, const MxProblem& g, int* tile_n, int* pair) {
    const int64_t n = (g.N + g.groups - 1) / g.groups;
    *tile_n = h->tile_n ? std::max(h->tile_n, 128) : n > 128 ? 256 : n > 32 ? 128 : 32;
    if (*tile_n == 256 && (g.M <= 128 || h->cta_pair == 1)) *tile_n = 128;
    if (*tile_n == 256) {
        const int64_t units = (g.M + 255) / 256 * (g.N / 256 + std::min(g.groups, g.N));
        if (g.beta != 0.0f ? (g.K <= 2048 || units <= h->sm_count) : g.K <= 512) *tile_n = 192;
    }
    *pair = *tile_n >= 192 ? 2 : 1;
}

int run(b200_handle* h, cudaStream_t stream, const MxProblem& g) {
    int tile_n, pair, rc;
    pick_tile(h, g, &tile_n, &pair);
    MxGemmParams p = {};
    p.N = static_cast<int>(g.N);
    p.K = static_cast<int>(g.K);
    p.groups = static_cast<int>(g.groups);
    const int64_t tiles_m = (g.M + 128 * pair - 1) / (128 * pair);
    p.raster = Raster::of(h->raster_group > 0 ? h->raster_group : 8, static_cast<int>(tiles_m));
    p.offsets = g.offsets;
    p.a_per_group = g.stride_a != 0 ? 1 : 0;
    p.a_tile_rows = static_cast<int>((g.M + 127) / 128);
    p.e.M = static_cast<int>(g.M);
    p.e.alpha = g.alpha;
    p.e.beta = g.beta;
    p.e.C = g.C;
    p.e.D = g.D;
    p.e.ldc = g.ldc;
    p.e.ldd = g.ldd;
    p.e.c_fmt = elem_fmt(g.c_type);
    p.e.d_fmt = elem_fmt(g.d_type);
    p.e.whole_kb = mx_whole_kb(p.e.d_fmt);
    p.status = h->status_word;
    p.wait_budget_ns = h->wait_budget_ns;
    p.e.d_pairs = !(reinterpret_cast<uintptr_t>(g.D) & 3u) && g.ldd % 2 == 0;

    const int bn_local = tile_n / pair, bbox = std::min(bn_local, 128);
    const int64_t k_bytes = (g.K + 1) / 2;
    CUtensorMap tm[4];
    BatchDim b;
    b.count = g.stride_a != 0 ? g.groups : 1;
    b.stride = b.count > 1 ? g.stride_a / 2 : g.lda / 2 * g.M;
    if ((rc = encode_map_2d(&tm[0], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.A, k_bytes, g.M, g.lda / 2, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B, "A", b))) return rc;
    if ((rc = encode_map_2d(&tm[1], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.B, k_bytes, g.N, g.ldb / 2, 128, bbox, CU_TENSOR_MAP_SWIZZLE_128B, "B"))) return rc;
    // scales: tiles of 128 words, K tiles, rows of tiles; a copy takes 2 along K.  How many rows the groups of B use is not
    // known here, only the most they can: those copies take one row each
    const int64_t kt = (g.K + 127) / 128, sa_rows = p.a_tile_rows * b.count;
    const int64_t sb_rows = b200_mxfp4_scale_bytes(g.K, g.N, g.offsets ? g.groups : 0) / 512 / kt;
    if (sa_rows > 0x7fffff00ll || sb_rows > 0x7fffff00ll) return fail(B200_UNSUPPORTED, "mxfp4 gemm: too many scale tiles");
    auto scale_map = [&](CUtensorMap* m, const void* ptr, int64_t rows, int box_rows, const char* what) {
        BatchDim d;
        d.count = rows;
        d.stride = kt * 128;
        d.box = box_rows;
        return encode_map_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, ptr, 128, kt, 128, 128, 2, CU_TENSOR_MAP_SWIZZLE_NONE, what, d);
    };
    if ((rc = scale_map(&tm[2], g.SA, sa_rows, 1, "scales of A")) || (rc = scale_map(&tm[3], g.SB, sb_rows, g.offsets ? 1 : (tile_n + 127) / 128, "scales of B"))) return rc;
    const int64_t units = (g.N / tile_n + std::min(g.groups, g.N)) * tiles_m;
    if (units > 0x7fffff00ll) return fail(B200_UNSUPPORTED, "mxfp4 gemm: too many tiles for one launch");
    const int cap = h->max_ctas > 0 ? std::min(h->max_ctas, h->sm_count) : h->sm_count;
    int grid = static_cast<int>(std::min<int64_t>(std::max(cap / pair, 1), units)) * pair;
    if (tile_n == 32) grid = std::max(cap / 2, 1) * 2;  // pairs of CTAs; how many tiles there are is not known here
    const bool pdl = h->pdl != 0;
    if (tile_n == 256) rc = launch<256, 2>(tm, p, grid, stream, pdl);
    else if (tile_n == 192) rc = launch<192, 2>(tm, p, grid, stream, pdl);
    else if (tile_n == 128) rc = launch<128, 1>(tm, p, grid, stream, pdl);
    else rc = launch<32, 1>(tm, p, grid, stream, pdl);
    if (rc) return rc;
    h->last = {B200_KERNEL_TCGEN05, tile_n, 1, grid, pair};
    return B200_OK;
}

bool is_elem_type(int t) { return t == B200_F16 || t == B200_F32 || t == B200_BF16; }

int entry(b200_handle* h, cudaStream_t stream, const MxProblem& g) {
    auto bad = [&](const char* m) { return fail(B200_INVALID_ARG, std::string("mxfp4 gemm: ") + m); };
    const int64_t most = 0x7fffff00ll, k32 = (g.K + 31) / 32 * 32;
    if (!is_elem_type(g.c_type) || !is_elem_type(g.d_type)) return bad("C and D must be Float16, bfloat16 or Float32");
    if (g.M < 0 || g.N < 0 || g.K < 0) return bad("negative dimension");
    if (g.M > most || g.N > most || g.K > most) return bad("dimension exceeds 2^31");
    if (g.groups < 0 || g.groups > kMaxGroups) return bad("groups must be in [0, 1024]");
    if (g.lda < k32 || g.ldb < k32 || g.lda % 32 || g.ldb % 32) return bad("lda and ldb must be multiples of 32 and at least K rounded up to 32");
    if (g.stride_a < 0 || g.stride_a % 32) return bad("stride_a must be a multiple of 32");
    if (g.groups > 1 && g.stride_a != 0 && g.stride_a < g.lda * g.M) return bad("stride_a smaller than one matrix");
    if (g.ldd < std::max<int64_t>(1, g.M)) return bad("ldd smaller than M");
    if (g.beta != 0.0f && g.ldc < std::max<int64_t>(1, g.M)) return bad("ldc smaller than M");
    if (g.M == 0 || g.N == 0 || g.groups == 0) return B200_OK;
    if (g.K == 0) return bad("K must be positive");
    if (!g.A || !g.B || !g.SA || !g.SB) return bad("A, B or a scale pointer is null");
    if (!g.D) return bad("D is null");
    if (g.beta != 0.0f && !g.C) return bad("C is null but beta != 0");
    if ((reinterpret_cast<uintptr_t>(g.A) | reinterpret_cast<uintptr_t>(g.B) | reinterpret_cast<uintptr_t>(g.SA) | reinterpret_cast<uintptr_t>(g.SB)) & 15u)
        return bad("elements and scales must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(g.offsets) % 4 || reinterpret_cast<uintptr_t>(g.D) % elem_bytes(g.d_type) ||
        (g.beta != 0.0f && reinterpret_cast<uintptr_t>(g.C) % elem_bytes(g.c_type)))
        return bad("a pointer is not aligned to its element type");
    if (h->force_kernel == B200_KERNEL_SIMPLE) return fail(B200_UNSUPPORTED, "mxfp4 gemm: there is no simple kernel for 4-bit operands");
    int rc;
    if ((rc = poll_previous_launch(h)) || (rc = check_current_device(h))) return rc;
    rc = run(h, stream, g);
    return rc ? rc : note_launch(h, stream);
}

}  // namespace
}  // namespace b200

extern "C" int b200_gemm_mxfp4(b200_handle* h, b200_stream stream, int64_t M, int64_t N, int64_t K, float alpha, const void* A, int64_t lda,
                               const void* a_scales, const void* B, int64_t ldb, const void* b_scales, float beta, const void* C, int64_t ldc,
                               int c_type, void* D, int64_t ldd, int d_type) {
    if (!h) return b200::fail(B200_INVALID_ARG, "null handle");
    const b200::MxProblem g = {M, N, K, 1, alpha, beta, A, a_scales, B, b_scales, C, D, lda, 0, ldb, ldc, ldd, c_type, d_type, nullptr};
    return b200::entry(h, static_cast<cudaStream_t>(stream), g);
}

extern "C" int b200_gemm_mxfp4_grouped(b200_handle* h, b200_stream stream, int64_t M, int64_t N, int64_t K, float alpha, const void* A, int64_t lda,
                                       int64_t stride_a, const void* a_scales, const void* B, int64_t ldb, const void* b_scales, float beta,
                                       const void* C, int64_t ldc, int c_type, void* D, int64_t ldd, int d_type, const int32_t* offsets,
                                       int64_t groups) {
    if (!h) return b200::fail(B200_INVALID_ARG, "null handle");
    if (!offsets && groups > 0 && M > 0 && N > 0) return b200::fail(B200_INVALID_ARG, "mxfp4 gemm: offsets is null");
    const b200::MxProblem g = {M, N, K, groups, alpha, beta, A, a_scales, B, b_scales, C, D, lda, stride_a, ldb, ldc, ldd, c_type, d_type, offsets};
    return b200::entry(h, static_cast<cudaStream_t>(stream), g);
}
