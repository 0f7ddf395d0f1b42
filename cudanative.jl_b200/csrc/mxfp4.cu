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

// 32 values -> scale code and elements.
__device__ __forceinline__ uint32_t quantize_block(float (&v)[32], uint4* q) {
    uint32_t top = 0;  // binary32 magnitudes order like integers
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t e = top >> 23;  // biased exponent; 0 for zero and subnormals
    const uint32_t s = e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
    const float inv = __uint_as_float((e == 255 ? 0u : 254u - s) << 23);  // 2^(127 - s), normal for every s <= 252
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= inv;
    *q = make_uint4(to_elements(v), to_elements(v + 8), to_elements(v + 16), to_elements(v + 24));
    return s;
}

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

// One block of 32 values per thread.  kTrans = 0: a vector's values are contiguous, four neighbouring
// threads take four blocks of one vector (and write its four scales as one word); kTrans = 1: vectors are
// contiguous across, a warp takes one block of 32 vectors.
template <typename T, bool kTrans>
__global__ void __launch_bounds__(256) mxfp4_quantize_kernel(const MxParams p) {
    __shared__ int off[kMaxGroups + 1], first[kMaxGroups + 1], sums[8];
    long long tile_rows = (p.cols + 127) / 128;
    if (p.offsets) {
        if (!load_groups<true>(p.offsets, p.groups, p.cols, 128, off, first, sums)) {
            if (threadIdx.x == 0) atomicCAS(p.status, 0, static_cast<int>(kBadOffsets));
            return;
        }
        tile_rows = first[p.groups];
    }
    const int kt = (p.K + 127) / 128;
    const T* X = static_cast<const T*>(p.X);
    const long long work = tile_rows * kt;  // a tile of 128 vectors x 128 values: 512 blocks, two per thread
    for (long long w = blockIdx.x; w < work; w += gridDim.x) {
        const long long q = w / kt;
        const int k_tile = static_cast<int>(w - q * kt);
        const TileRow t = tile_row(p, off, first, q);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            const int i = threadIdx.x + half * 256;
            const int r = kTrans ? (i & 31) + (i >> 7) * 32 : i >> 2;
            const int b = kTrans ? (i >> 5) & 3 : i & 3;
            const int k0 = k_tile * 128 + b * 32;
            uint32_t s = 0;
            if (r < t.count && k0 < p.K) {
                const long long vec = t.first + r;
                float v[32];
                const T* src = kTrans ? X + vec + static_cast<long long>(k0) * p.ldx : X + vec * p.ldx + k0;
                const long long step = kTrans ? p.ldx : 1;
                constexpr int kVec = 16 / sizeof(T);
                if (!kTrans && k0 + 32 <= p.K && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
                    for (int j = 0; j < 32 / kVec; ++j) {
                        const uint4 raw = reinterpret_cast<const uint4*>(src)[j];
                        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
                        for (int x = 0; x < kVec; ++x) v[j * kVec + x] = as_float(e[x]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = k0 + j < p.K ? as_float(src[j * step]) : 0.0f;
                }
                uint4 elements;
                s = quantize_block(v, &elements);
                *reinterpret_cast<uint4*>(p.Q + (vec * p.ldq + k0) / 2) = elements;
            }
            if constexpr (kTrans) {
                p.S[scale_at(q, kt, k_tile * 4 + b, r)] = static_cast<uint8_t>(s);
            } else {
                s <<= 8 * b;
                s |= __shfl_xor_sync(0xffffffffu, s, 1);
                s |= __shfl_xor_sync(0xffffffffu, s, 2);
                if (b == 0) *reinterpret_cast<uint32_t*>(p.S + scale_at(q, kt, k_tile * 4, r)) = s;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) mxfp4_dequantize_kernel(const MxParams p) {
    __shared__ int off[kMaxGroups + 1], first[kMaxGroups + 1], sums[8];
    long long tile_rows = (p.cols + 127) / 128;
    if (p.offsets) {
        if (!load_groups<true>(p.offsets, p.groups, p.cols, 128, off, first, sums)) {
            if (threadIdx.x == 0) atomicCAS(p.status, 0, static_cast<int>(kBadOffsets));
            return;
        }
        tile_rows = first[p.groups];
    }
    const int kt = (p.K + 127) / 128;
    T* Y = static_cast<T*>(p.Y);
    const long long work = tile_rows * kt;
    for (long long w = blockIdx.x; w < work; w += gridDim.x) {
        const long long q = w / kt;
        const int k_tile = static_cast<int>(w - q * kt);
        const TileRow t = tile_row(p, off, first, q);
        // eight elements (4 bytes) per thread and step: 16 threads to a vector's 128
#pragma unroll 2
        for (int i = threadIdx.x; i < 128 * 16; i += 256) {
            const int r = i >> 4, k0 = k_tile * 128 + (i & 15) * 8;
            if (r >= t.count || k0 >= p.K) continue;
            const long long vec = t.first + r;
            const uint32_t bits = *reinterpret_cast<const uint32_t*>(p.Q + (vec * p.ldq + k0) / 2);
            const uint32_t s = p.S[scale_at(q, kt, k0 / 32, r)];
            const float x = __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23);
            T out[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t c = (bits >> (4 * j)) & 15u, m = c & 7u;
                // magnitude: 0, .5, then (1 + .5 f) 2^(e - 1) with e = m >> 1, f = m & 1
                const float a = m < 2 ? 0.5f * m : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
                out[j] = from_float<T>((c & 8u ? -a : a) * x);
            }
            T* dst = Y + vec * p.ldy + k0;
            if (k0 + 8 <= p.K && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
                for (int j = 0; j < static_cast<int>(8 * sizeof(T) / 16); ++j)
                    reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(out)[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + j < p.K) dst[j] = out[j];
            }
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

int grid_for(const b200_handle* h, int64_t K, int64_t cols, int64_t groups) {
    const int64_t tiles = (cols / 128 + std::max<int64_t>(1, std::min(groups, cols))) * ((K + 127) / 128);
    return static_cast<int>(std::min<int64_t>(tiles, static_cast<int64_t>(h->sm_count) * 8));
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
    const int grid = grid_for(h, K, cols, groups);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define B200_QUANTIZE(T)                                                    \
    do {                                                                    \
        if (trans) mxfp4_quantize_kernel<T, true><<<grid, 256, 0, st>>>(p); \
        else mxfp4_quantize_kernel<T, false><<<grid, 256, 0, st>>>(p);      \
    } while (0)
    if (x_type == B200_F32) B200_QUANTIZE(float);
    else if (x_type == B200_F16) B200_QUANTIZE(__half);
    else B200_QUANTIZE(__nv_bfloat16);
#undef B200_QUANTIZE
    B200_CUDA_TRY(cudaGetLastError());
    return note_launch(h, st);
}

extern "C" int b200_mxfp4_dequantize(b200_handle* h, b200_stream stream, int64_t K, int64_t cols, const void* Q, int64_t ldq, const void* S, void* Y,
                                     int64_t ldy, int y_type, const int32_t* offsets, int64_t groups) {
    if (!h) return fail(B200_INVALID_ARG, "null handle");
    int rc = check_mx("mxfp4_dequantize", K, cols, groups, Y, ldy, K, y_type, Q, ldq, S, offsets);
    if (rc || K == 0 || cols == 0) return rc;
    if ((rc = poll_previous_launch(h)) || (rc = check_current_device(h))) return rc;
    const MxParams p = {nullptr, 0, const_cast<uint8_t*>(static_cast<const uint8_t*>(Q)), ldq, const_cast<uint8_t*>(static_cast<const uint8_t*>(S)),
                        Y, ldy, static_cast<int>(K), static_cast<int>(cols), static_cast<int>(groups), offsets, h->status_word};
    const int grid = grid_for(h, K, cols, groups);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (y_type == B200_F32) mxfp4_dequantize_kernel<float><<<grid, 256, 0, st>>>(p);
    else if (y_type == B200_F16) mxfp4_dequantize_kernel<__half><<<grid, 256, 0, st>>>(p);
    else mxfp4_dequantize_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
    B200_CUDA_TRY(cudaGetLastError());
    return note_launch(h, st);
}
