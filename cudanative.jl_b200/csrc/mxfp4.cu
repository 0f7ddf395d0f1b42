// Microscaled 4-bit values: quantisation and its inverse.
//
// A block of 32 values along K shares a power of two, X = 2^(s - 127) with an 8-bit code s; each value is
// a 4-bit element (sign, 2 exponent bits, 1 fraction bit: 0, .5, 1, 1.5, 2, 3, 4, 6).  Quantising takes
// X = 2^(floor(log2(max |v|)) - 2), the largest power for which the block's largest value is below twice
// the largest element's binade, and rounds v / X to the nearest element, ties to even, saturating at 6.
// v / X is exact in binary32 (a power of two), so the result is the correctly rounded one.  A block that
// holds a NaN or an infinity gets s = 255, which stands for NaN, and the whole block reads as NaN.
//
// Scales lie where the tensor core's block-scaled product wants them: tiles of 512 bytes for 128 vectors
// x 4 blocks, vector r and block b of a tile at byte (r % 32) * 16 + (r / 32) * 4 + b; the tiles of one
// 128 vectors follow each other along K.  All of a tile is written, 0 (2^-127) where there is no block.
//
// Both kernels are bound by memory: per value 2 (4) bytes in and 17/32 out, or the other way round.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "gemm_grouped.cuh"
#include "internal.h"

namespace b200 {
namespace {

struct MxParams {
    const void* X;
    long long ldx;
    uint8_t* Q;
    long long ldq;  // elements
    uint8_t* S;
    void* Y;
    long long ldy;
    int K, cols, groups;
    const int* offsets;
    int* status;
};

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <> __device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// Eight values -> eight 4-bit elements, the first in the lowest four bits.
__device__ __forceinline__ uint32_t to_elements(const float* v) {
    uint32_t r;
    asm("{\n"
        ".reg .b8 t0, t1, t2, t3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n"
        "mov.b32 %0, {t0, t1, t2, t3};\n"
        "}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Eight elements times x.
template <typename T>
__device__ __forceinline__ void from_elements(uint32_t bits, float x, T (&out)[8]) {
    uint32_t h[4];  // two binary16 each: every element is exact in it
    asm("{\n"
        ".reg .b8 t0, t1, t2, t3;\n"
        "mov.b32 {t0, t1, t2, t3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, t0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, t1;\n"
        "cvt.rn.f16x2.e2m1x2 %2, t2;\n"
        "cvt.rn.f16x2.e2m1x2 %3, t3;\n"
        "}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(bits));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        out[2 * j] = from_float<T>(v.x * x);
        out[2 * j + 1] = from_float<T>(v.y * x);
    }
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // orders like the values

// Scale code of a block whose largest magnitude is `top` (binary32 bits).
__device__ __forceinline__ uint32_t scale_code(uint32_t top) {
    const uint32_t e = top >> 23;  // biased exponent; 0 for zero and subnormals
    return e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
}

// 1 / X = 2^(127 - s), a normal number for every s <= 252; 0 for a block of NaN.
__device__ __forceinline__ float inverse(uint32_t s) { return __uint_as_float((s == 255 ? 0u : 254u - s) << 23); }

__device__ __forceinline__ long long scale_at(long long tile_row, int kt, int kblock, int r) {
    return (tile_row * kt + kblock / 4) * 512 + (r % 32) * 16 + (r / 32) * 4 + kblock % 4;
}

// The vectors of scale tile row q: first vector and how many of the 128 exist.
struct TileRow {
    long long first;
    int count;
};
__device__ __forceinline__ TileRow tile_row(const MxParams& p, const int* off, const int* first, long long q) {
    if (!p.offsets) return {q * 128, static_cast<int>(min(128ll, p.cols - q * 128))};
    const int e = find_group(first, p.groups, static_cast<int>(q));
    const long long v0 = off[e] + (q - first[e]) * 128ll;
    return {v0, static_cast<int>(min(128ll, off[e + 1] - v0))};
}

// What every block of a launch needs: the groups' rows of scale tiles, and how many there are; 0 for bad offsets.
__device__ __forceinline__ long long scale_tile_rows(const MxParams& p, int* off, int* first, unsigned long long* sums) {
    if (!p.offsets) return (p.cols + 127) / 128;
    if (!load_groups<true>(p.offsets, p.groups, p.cols, 128, off, first, sums)) {
        if (threadIdx.x == 0) report_bad_offsets(p.status, p.groups);
        return 0;
    }
    return first[p.groups];
}

// Vectors whose values are contiguous.  A tile is 128 vectors x 128 values: 16 lanes take a vector's 128, eight
// values (16 bytes of a 16-bit type) each, so that a warp reads and writes whole lines; four lanes find a
// block's largest magnitude with two shuffles.  A thread has four vectors in flight, four blocks share an SM: Float16
// 16384 x 2048 19.0 us (4.5 TB/s; three blocks 20.6, five 20.3; eight vectors and three blocks 22.7).
template <typename T>
__global__ void __launch_bounds__(256, 4) mxfp4_quantize_kernel(const MxParams p) {
    __shared__ int off[kMaxGroups + 1], first[kMaxGroups + 1];
    __shared__ unsigned long long sums[8];
    griddep_launch_dependents();
    griddep_wait();
    const long long tile_rows = scale_tile_rows(p, off, first, sums);
    const int kt = (p.K + 127) / 128;
    const T* X = static_cast<const T*>(p.X);
    const long long work = tile_rows * kt;
    const int lane = threadIdx.x & 31, part = lane & 15;
    const int first_row = (threadIdx.x >> 5) * 2 + (lane >> 4);
    const bool wide = p.ldx % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(X) & 15u) == 0;
    for (long long w = blockIdx.x; w < work; w += gridDim.x) {
        const long long q = w / kt;
        const int k_tile = static_cast<int>(w - q * kt);
        const TileRow t = tile_row(p, off, first, q);
        const int k0 = k_tile * 128 + part * 8;
        constexpr int kVec = 8 * sizeof(T) / 16;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            const int r0 = first_row + 64 * half;
            uint4 raw[4][kVec];
            const T* src = X + (t.first + r0) * p.ldx + k0;
            if (wide && k_tile * 128 + 128 <= p.K) {  // all loads before the first use
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kVec; ++j)
                        raw[i][j] = r0 + 16 * i < t.count ? reinterpret_cast<const uint4*>(src + 16 * i * p.ldx)[j] : make_uint4(0, 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    T* e = reinterpret_cast<T*>(raw[i]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = r0 + 16 * i < t.count && k0 + j < p.K ? src[16 * i * p.ldx + j] : from_float<T>(0.0f);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = r0 + 16 * i;
                const T* e = reinterpret_cast<const T*>(raw[i]);
                float v[8];
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = as_float(e[j]);
                    top = max(top, magnitude(v[j]));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                uint32_t s = scale_code(top);
                const float inv = inverse(s);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= inv;
                if (r < t.count && k0 < (p.K + 31) / 32 * 32) *reinterpret_cast<uint32_t*>(p.Q + ((t.first + r) * p.ldq + k0) / 2) = to_elements(v);
                // a vector's four scales as one word; vectors and blocks that do not exist were read as zeros: s = 0
                s <<= 8 * (part / 4);
                s |= __shfl_xor_sync(0xffffffffu, s, 4);
                s |= __shfl_xor_sync(0xffffffffu, s, 8);
                if (part == 0) *reinterpret_cast<uint32_t*>(p.S + scale_at(q, kt, k_tile * 4, r)) = s;
            }
        }
    }
}

// Vectors that lie across (X is cols x K): a thread takes one block of two neighbouring vectors, so that a warp
// reads 64 vectors' values of one k as a line; elements and scales of the tile go out through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) mxfp4_quantize_across_kernel(const MxParams p) {
    __shared__ int off[kMaxGroups + 1], first[kMaxGroups + 1];
    __shared__ unsigned long long sums[8];
    __shared__ __align__(16) uint8_t elements[128][64 + 16];
    __shared__ __align__(16) uint8_t scales[512];
    griddep_launch_dependents();
    griddep_wait();
    const long long tile_rows = scale_tile_rows(p, off, first, sums);
    const int kt = (p.K + 127) / 128;
    const T* X = static_cast<const T*>(p.X);
    const long long work = tile_rows * kt;
    const int r = (threadIdx.x & 63) * 2, b = threadIdx.x >> 6;
    struct alignas(2 * sizeof(T)) Pair { T a, b; };
    for (long long w = blockIdx.x; w < work; w += gridDim.x) {
        const long long q = w / kt;
        const int k_tile = static_cast<int>(w - q * kt);
        const TileRow t = tile_row(p, off, first, q);
        const int k0 = k_tile * 128 + b * 32;
        const T* src = X + t.first + r + static_cast<long long>(k0) * p.ldx;
        const bool pairs = p.ldx % 2 == 0 && (reinterpret_cast<uintptr_t>(src) % sizeof(Pair)) == 0;
        Pair raw[32];
        if (pairs && r + 1 < t.count && k0 + 32 <= p.K) {  // all loads before the first use
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = *reinterpret_cast<const Pair*>(src + j * p.ldx);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                raw[j].a = r < t.count && k0 + j < p.K ? src[j * p.ldx] : from_float<T>(0.0f);
                raw[j].b = r + 1 < t.count && k0 + j < p.K ? src[j * p.ldx + 1] : from_float<T>(0.0f);
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) top = max(top, magnitude(as_float(x ? raw[j].b : raw[j].a)));
            const uint32_t s = scale_code(top);
            const float inv = inverse(s);
            uint32_t e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = as_float(x ? raw[i * 8 + j].b : raw[i * 8 + j].a) * inv;
                e[i] = to_elements(v);
            }
            *reinterpret_cast<uint4*>(&elements[r + x][b * 16]) = make_uint4(e[0], e[1], e[2], e[3]);
            scales[((r + x) % 32) * 16 + (r + x) / 32 * 4 + b] = static_cast<uint8_t>(s);
        }
        __syncthreads();
#pragma unroll
        for (int i = threadIdx.x; i < 512; i += 256) {
            const int row = i >> 2, part = i & 3;
            const int k = k_tile * 128 + part * 32;
            if (row < t.count && k < p.K)
                *reinterpret_cast<uint4*>(p.Q + ((t.first + row) * p.ldq + k) / 2) = *reinterpret_cast<const uint4*>(&elements[row][part * 16]);
        }
        if (threadIdx.x < 32)
            reinterpret_cast<uint4*>(p.S + (q * kt + k_tile) * 512)[threadIdx.x] = reinterpret_cast<const uint4*>(scales)[threadIdx.x];
        __syncthreads();
    }
}

// Eight elements to a thread, 16 lanes to a vector's 128, eight vectors in flight.  Binary32 rows, and rows of Y
// that do not begin on 16 bytes, are put together in shared memory and leave lane next to lane, 16 bytes, 4 or
// single values each.  Four blocks per SM: 8192 x 8192 to bfloat16 32 us (5.3 TB/s; three 36, five 39 us).
template <typename T>
__global__ void __launch_bounds__(256, 4) mxfp4_dequantize_kernel(const MxParams p) {
    __shared__ int off[kMaxGroups + 1], first[kMaxGroups + 1];
    __shared__ unsigned long long sums[8];
    __shared__ __align__(16) T rows[16][128 + 16 / sizeof(T)];
    griddep_launch_dependents();
    griddep_wait();
    const long long tile_rows = scale_tile_rows(p, off, first, sums);
    const int kt = (p.K + 127) / 128;
    T* Y = static_cast<T*>(p.Y);
    const long long work = tile_rows * kt;
    const int lane = threadIdx.x & 31, part = lane & 15, r0 = (threadIdx.x >> 5) * 2 + (lane >> 4);
    const bool wide = p.ldy % (16 / sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(Y) & 15u) == 0;
    const bool words = p.ldy * sizeof(T) % 4 == 0 && (reinterpret_cast<uintptr_t>(Y) & 3u) == 0;
    for (long long w = blockIdx.x; w < work; w += gridDim.x) {
        const long long q = w / kt;
        const int k_tile = static_cast<int>(w - q * kt);
        const TileRow t = tile_row(p, off, first, q);
        const int k0 = k_tile * 128 + part * 8;
        uint32_t bits[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + 16 * i;
            const bool there = r < t.count && k0 < p.K;
            bits[i] = there ? *reinterpret_cast<const uint32_t*>(p.Q + ((t.first + r) * p.ldq + k0) / 2) : 0u;
            s[i] = there ? p.S[scale_at(q, kt, k_tile * 4 + part / 4, r)] : 0u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + 16 * i;
            const float x = __uint_as_float(s[i] == 0 ? 0x00400000u : s[i] == 255 ? 0x7fc00000u : s[i] << 23);
            alignas(16) T out[8];
            from_elements(bits[i], x, out);
            constexpr int kVec = 8 * sizeof(T) / 16;
            const bool full = wide && k_tile * 128 + 128 <= p.K;
            if (full && sizeof(T) == 2) {
                if (r < t.count) {
#pragma unroll
                    for (int j = 0; j < kVec; ++j) reinterpret_cast<uint4*>(Y + (t.first + r) * p.ldy + k0)[j] = reinterpret_cast<const uint4*>(out)[j];
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < kVec; ++j) reinterpret_cast<uint4*>(&rows[r0][part * 8])[j] = reinterpret_cast<const uint4*>(out)[j];
            __syncwarp();
            const int n = min(128, p.K - k_tile * 128);
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {  // the warp's two vectors
                const int rr = (threadIdx.x >> 5) * 2 + x2;
                if (rr + 16 * i >= t.count) continue;
                T* dst = Y + (t.first + rr + 16 * i) * p.ldy + k_tile * 128;
                if (full) {  // binary32: a lane's own eight values are two halves of different lines of stores
                    reinterpret_cast<uint4*>(dst)[lane] = *reinterpret_cast<const uint4*>(&rows[rr][lane * (16 / sizeof(T))]);
                } else if (words && sizeof(T) == 2 && n % 2 == 0) {
#pragma unroll
                    for (int j = lane * 2; j < 128; j += 64)
                        if (j < n) *reinterpret_cast<uint32_t*>(dst + j) = *reinterpret_cast<const uint32_t*>(&rows[rr][j]);
                } else {
                    for (int j = lane; j < n; j += 32) dst[j] = rows[rr][j];
                }
            }
            __syncwarp();
        }
    }
}

bool is_elem_type(int t) { return t == B200_F16 || t == B200_F32 || t == B200_BF16; }

int check_mx(const char* what, int64_t K, int64_t cols, int64_t groups, const void* values, int64_t ld, int64_t ld_min, int type, const void* Q,
             int64_t ldq, const void* S, const int32_t* offsets) {
    const std::string name = std::string(what) + ": ";
    auto bad = [&](const char* m) { return fail(B200_INVALID_ARG, name + m); };
    if (!is_elem_type(type)) return bad("values must be Float16, bfloat16 or Float32");
    if (K < 0 || cols < 0) return bad("negative dimension");
    if (K > 0x7fffff00ll || cols > 0x7fffff00ll) return bad("dimension exceeds 2^31");
    if (ld < std::max<int64_t>(1, ld_min)) return bad("leading dimension of the values too small");
    if (ldq < (K + 31) / 32 * 32 || ldq % 32) return bad("ldq must be a multiple of 32 and at least K rounded up to 32");
    if (groups < 0 || groups > kMaxGroups) return bad("groups must be in [0, 1024]");
    if (offsets ? groups == 0 : groups != 0) return bad("offsets and groups go together");
    if (K == 0 || cols == 0) return B200_OK;
    if (!values || !Q || !S) return bad("a pointer is null");
    if (reinterpret_cast<uintptr_t>(values) % elem_bytes(type) || reinterpret_cast<uintptr_t>(offsets) % 4)
        return bad("a pointer is not aligned to its element type");
    if ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(S)) & 15u) return bad("elements and scales must be 16-byte aligned");
    return B200_OK;
}

int launch_mx(const b200_handle* h, void (*kern)(MxParams), const MxParams& p, cudaStream_t stream) {
    const int64_t tiles = (p.cols / 128 + std::max<int64_t>(1, std::min(p.groups, p.cols))) * ((p.K + 127) / 128);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tiles, static_cast<int64_t>(h->sm_count) * 8)), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = h->pdl ? 1 : 0;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int64_t b200_mxfp4_scale_bytes(int64_t K, int64_t cols, int64_t groups) {
    if (K < 0 || cols < 0 || groups < 0) return 0;
    const int64_t rows = groups > 0 ? (cols + 127 * std::min(groups, cols)) / 128 : (cols + 127) / 128;
    return rows * ((K + 127) / 128) * 512;
}

extern "C" int b200_mxfp4_quantize(b200_handle* h, b200_stream stream, int trans, int64_t K, int64_t cols, const void* X, int64_t ldx, int x_type,
                                   void* Q, int64_t ldq, void* S, const int32_t* offsets, int64_t groups) {
    if (!h) return fail(B200_INVALID_ARG, "null handle");
    if (trans != 0 && trans != 1) return fail(B200_INVALID_ARG, "mxfp4_quantize: trans must be 0 or 1");
    int rc = check_mx("mxfp4_quantize", K, cols, groups, X, ldx, trans ? cols : K, x_type, Q, ldq, S, offsets);
    if (rc || K == 0 || cols == 0) return rc;
    if ((rc = poll_previous_launch(h)) || (rc = check_current_device(h))) return rc;
    const MxParams p = {X, ldx, static_cast<uint8_t*>(Q), ldq, static_cast<uint8_t*>(S), nullptr, 0, static_cast<int>(K), static_cast<int>(cols),
                        static_cast<int>(groups), offsets, h->status_word};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (x_type == B200_F32) rc = launch_mx(h, trans ? mxfp4_quantize_across_kernel<float> : mxfp4_quantize_kernel<float>, p, st);
    else if (x_type == B200_F16) rc = launch_mx(h, trans ? mxfp4_quantize_across_kernel<__half> : mxfp4_quantize_kernel<__half>, p, st);
    else rc = launch_mx(h, trans ? mxfp4_quantize_across_kernel<__nv_bfloat16> : mxfp4_quantize_kernel<__nv_bfloat16>, p, st);
    return rc ? rc : note_launch(h, st);
}

extern "C" int b200_mxfp4_dequantize(b200_handle* h, b200_stream stream, int64_t K, int64_t cols, const void* Q, int64_t ldq, const void* S, void* Y,
                                     int64_t ldy, int y_type, const int32_t* offsets, int64_t groups) {
    if (!h) return fail(B200_INVALID_ARG, "null handle");
    int rc = check_mx("mxfp4_dequantize", K, cols, groups, Y, ldy, K, y_type, Q, ldq, S, offsets);
    if (rc || K == 0 || cols == 0) return rc;
    if ((rc = poll_previous_launch(h)) || (rc = check_current_device(h))) return rc;
    const MxParams p = {nullptr, 0, const_cast<uint8_t*>(static_cast<const uint8_t*>(Q)), ldq, const_cast<uint8_t*>(static_cast<const uint8_t*>(S)),
                        Y, ldy, static_cast<int>(K), static_cast<int>(cols), static_cast<int>(groups), offsets, h->status_word};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (y_type == B200_F32) rc = launch_mx(h, mxfp4_dequantize_kernel<float>, p, st);
    else if (y_type == B200_F16) rc = launch_mx(h, mxfp4_dequantize_kernel<__half>, p, st);
    else rc = launch_mx(h, mxfp4_dequantize_kernel<__nv_bfloat16>, p, st);
    return rc ? rc : note_launch(h, st);
}
