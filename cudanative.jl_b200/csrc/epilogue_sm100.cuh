// Epilogue shared by the grouped and the 4-bit products: D = alpha * acc + beta * C from accumulators in
// tensor memory, by two groups of four warps, each with one half of a tile's columns.
//
// Why two groups: with short inner dimensions (a group's tokens, four-bit operands) a tile's main loop
// takes as long as reading its accumulator.
//
// A thread holds one row; D is column-major, so a warp's 32 rows of a column are one contiguous piece: 128
// bytes of a binary32 D, which go out as they are, and 64 of a 16-bit one, where neighbouring lanes
// exchange values so that each stores two rows at once.  No chunk passes through shared memory: staging
// for bulk stores took two barriers, a proxy fence and a copy's issue per 16 columns, 750 cycles (1 300 with C)
// where the stores themselves take about 100; it also cost 48 KiB of the ring.  Any M, leading dimension and
// alignment take the same path.
// With one k-block per tile the instructions of these warps are the bound: one uniform branch per 32 columns on the
// format and addresses that move on by addition took 256 groups of 512 x 768, 16 columns each, from 53 to 48 us
// (bfloat16 D; 42 us for the stores alone) and from 81 to 77 us (Float32).  All of a tile's accumulator at once, its four steps
// unrolled, was slower (70 us).
//
// C is read the same way: before it waits for the accumulator the warp brings the tile's lines of C into L2 and
// asks for the first step's values, then for each next step's while one is stored (where the registers
// allow it, kAhead).  32 groups of 2048 x 1408, 16384 columns, C and D Float32, loops of a few ms: 169 us (180-205 us in
// blocks of 0.15 s); 184 us without the values ahead, 203 us without the lines, 215 us with the lines of the next tile
// instead, 182 us with a ring of bulk copies of C in shared memory, which took 48 KiB from the stages (132 against 138 us
// without a C).
//
// kPromoteKb: the tensor core adds into its accumulator without rounding to nearest; every step drops what
// lies below the last place, which pulls sums towards zero in proportion to the number of steps (measured
// on K = 4096: 4e-6 of the result, 2e-5 for K = 16384; on K = 256 3e-7; on sums of one sign 1.1e-4 for K = 16384 and
// 1.7e-3 for 262144).  For a binary32 D that is more than the result's own precision, so the MMA issuer starts a new
// accumulator every kPromoteKb k-blocks and the warps add it, rounding to nearest, to a running sum in their
// registers while the next one is being filled.  A 16-bit D rounds by up to 2^-8 or 2^-11 of the result: it takes
// whole_kb k-blocks from one accumulator, which nearly always is all of K (kPromoteKb = 0), and kLong puts a longer sum
// together from several.
#pragma once

#include "ptx_sm100.cuh"

namespace b200 {

struct EpilogueParams {
    int M;
    float alpha, beta;
    const void* C;
    void* D;
    long long ldc, ldd, stride_c, stride_d;  // strides: one C and D per group (kPerGroup)
    int c_fmt, d_fmt;                        // 0 = binary32, 1 = binary16, 2 = bfloat16
    int whole_kb;                            // kLong: k-blocks that one accumulator sums at most, a power of two
    int d_pairs;                             // two rows of a 16-bit D can be stored as one word
};

// A tile of work: this CTA's first row, the tile's first column, the columns that exist; the inner dimension
// from k0 on, of which this CTA takes k-blocks (of 64 or 256) kb0 .. kb0 + kb - 1.
struct Unit {
    int group, m0, n0, cols, k0, k_len, kb0, kb;
};

// With few tiles the CTAs of a cluster share a tile's inner dimension.
// Two (kSplit = 2, few columns): CTA 1 sends its sums into CTA 0's shared memory, CTA 0 adds them to its own and
// stores.  Four (kSplit = 4, long inner dimension): the tile's 64 columns are dealt out, 16 to a CTA; every CTA sends each
// of the others its sums of the other's columns, adds what it gets for its own in the order of the CTAs, and stores.
constexpr int kSplitRow = 36;  // words per row of the receiver's buffer: 32 columns, and 4 against bank conflicts
struct SplitParams {
    int role = -1;       // -1: whole tiles, else this CTA's rank (of two: 0 receives and stores, 1 sends)
    const float* recv;   // two: [128][kSplitRow], four: [rank][128][16]
    uint32_t recv_addr;
    uint32_t full_bar, empty_bar;
};

template <int kBN>
struct EpilogueCfg {
    static constexpr int COLS = kBN >= 64 ? kBN / 2 : kBN;  // per warp group; the second is idle below 64
    static constexpr int W = 32;                            // columns per step
    static_assert(COLS % W == 0, "steps");
};

__device__ __forceinline__ int columns_of(int tile_cols, int wg, int cols) { return min(cols, max(0, tile_cols - wg * cols)); }

// Warps 4 .. 11 (`wg` 0 or 1).  Barriers tmem_full / tmem_empty [kAccs] are 8 bytes apart.
template <class E, int kBN, int kAccs, int kCtas, bool kF32, int kPromoteKb, bool kLong, bool kPerGroup, int kSplit, class Decode>
__device__ __forceinline__ void run_epilogue(const EpilogueParams& p, int wg, uint32_t tmem_base, uint32_t tmem_full, uint32_t tmem_empty,
                                             const WaitCtx& wc, int unit_first, int unit_stride, int num_units, const SplitParams& split,
                                             Decode decode) {
    constexpr int W = E::W;
    constexpr bool kDrain = kPromoteKb < 0;  // one accumulator: read it out at once so that the next tile may begin
    constexpr bool kAhead = !kDrain;
    const int et = static_cast<int>(threadIdx.x & 127);
    const int lane = static_cast<int>(threadIdx.x & 31);
    const uint32_t lane_base = static_cast<uint32_t>(((threadIdx.x >> 5) & 3) * 32) << 16;
    const bool has_c = p.beta != 0.0f;
    const float alpha = p.alpha, beta = p.beta;
    const int d_fmt = kF32 ? 0 : p.d_fmt;
    const int col0 = wg * E::COLS;
    uint32_t acc_count = 0, split_count = 0;
    bool ok = true;
    const bool sends = kSplit == 2 && split.role == 1, receives = kSplit == 2 && split.role == 0;
    const uint32_t remote = kSplit == 2 ? mapa_shared(split.recv_addr + et * kSplitRow * 4, 0) : 0u;
    const uint32_t remote_bar = kSplit == 2 ? mapa_shared(split.full_bar, 0) : 0u;
    static_assert(kSplit == 1 || (E::COLS == W && W == 32), "partial sums are one step of columns");

    // this warp's lines of C of a tile into L2, a lane to a column
    auto prefetch_c = [&](const Unit& u) {
        const int bytes = p.c_fmt == 0 ? 4 : 2, row = u.m0 + (et & ~31), cols = columns_of(u.cols, wg, E::COLS);
        for (int j = lane; j < cols; j += 32) {
            const long long at = (kPerGroup ? u.group * p.stride_c : 0) + row + (u.n0 + col0 + j) * p.ldc;
            if (row < p.M) asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(p.C) + at * bytes));
        }
    };

    for (int unit = unit_first; unit < num_units; unit += unit_stride) {
        const Unit u = decode(unit);
        const int cols = columns_of(u.cols, wg, E::COLS);
        const int m = u.m0 + et;
        const bool whole_rows = u.m0 + (et & ~31) + 32 <= p.M;  // of this warp

        // partial sums of the tile's columns, rounded up to four
        auto exchange = [&](uint32_t (&r)[W]) {
            if (sends) {
                ok = mbar_wait_cluster(split.empty_bar, (split_count & 1u) ^ 1u, wc, kWaitPartial);  // room over there
                ok = __all_sync(0xffffffffu, ok);
#pragma unroll
                for (int i = 0; i < W; i += 4)
                    if (ok && i < cols) st_async_cluster(remote + i * 4, r + i, remote_bar);
            } else {
                if (et == 0) mbar_arrive_expect_tx(split.full_bar, 128 * ((cols + 3) / 4 * 4) * 4);
                ok = mbar_wait_cluster(split.full_bar, split_count & 1u, wc, kWaitPartial);
                ok = __all_sync(0xffffffffu, ok);
                const float* in = split.recv + et * kSplitRow;
#pragma unroll
                for (int i = 0; i < W; i += 4) {
                    if (ok && i < cols) {
                        const float4 v = *reinterpret_cast<const float4*>(in + i);
                        r[i] = __float_as_uint(__uint_as_float(r[i]) + v.x);
                        r[i + 1] = __float_as_uint(__uint_as_float(r[i + 1]) + v.y);
                        r[i + 2] = __float_as_uint(__uint_as_float(r[i + 2]) + v.z);
                        r[i + 3] = __float_as_uint(__uint_as_float(r[i + 3]) + v.w);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(split.empty_bar, 1);
            }
            ++split_count;
        };
        // the accumulator has been read: the arrival carries no data, only that
        auto release = [&](uint32_t acc) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kCtas == 2) mbar_arrive_cluster_relaxed(tmem_empty + 8 * acc, 0);
                else mbar_arrive(tmem_empty + 8 * acc);
            }
        };
        auto wait_acc = [&](uint32_t acc) {
            ok = ok && mbar_wait(tmem_full + 8 * acc, (acc_count / kAccs) & 1u, wc, kWaitTmemFull);
            ok = __all_sync(0xffffffffu, ok);  // tcgen05.ld is warp-collective
            tc_fence_after_sync();
        };
        // Several accumulators: the last one takes the sum, and what follows finds it there.  The running
        // sums are indexed at run time and so lie in local memory: in registers they made the compiler spill in all of this
        // function, and short groups beside a long one took 22% longer (256 groups of 16 columns, 512 x 768: 51 -> 63 us).
        const bool longer = kLong && !kDrain && u.kb > p.whole_kb;
        if (longer) {
            float sum[E::COLS];
#pragma unroll 1
            for (int i = 0; i < E::COLS; ++i) sum[i] = 0.0f;
            for (int kb = 0; kb < u.kb; kb += p.whole_kb) {
                const uint32_t acc = acc_count % kAccs;
                const bool last = kb + p.whole_kb >= u.kb;
                wait_acc(acc);
                if (!ok) break;
#pragma unroll 1
                for (int q = 0; q < E::COLS; q += 16) {
                    if (q < cols) {
                        const uint32_t at = tmem_base + lane_base + acc * kBN + col0 + q;
                        uint32_t r[16];
                        tmem_ld_32x32b_x16(at, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[q + i] += __uint_as_float(r[i]);
                        if (last) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(sum[q + i]);
                            tmem_st_32x32b_x16(at, r);
                        }
                    }
                }
                if (last) break;
                release(acc);
                ++acc_count;
            }
            if (!ok) break;
            tmem_wait_st();
        }
        // C read directly: W columns ahead, the first before the accumulator is waited for, where the registers
        // are there for it (kAhead)
        float c_next[W];
        auto load_c = [&](int j) {
            const int left = cols - j * W;
            const long long at = (kPerGroup ? u.group * p.stride_c : 0) + m + (u.n0 + col0 + j * W) * p.ldc;
            if (p.c_fmt == 0) {
                const float* c = static_cast<const float*>(p.C) + at;
                if (whole_rows && left >= W) {
#pragma unroll
                    for (int i = 0; i < W; ++i) c_next[i] = c[i * p.ldc];
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) c_next[i] = m < p.M && i < left ? c[i * p.ldc] : 0.0f;
                }
            } else {
                const unsigned short* c = static_cast<const unsigned short*>(p.C) + at;
                unsigned short raw[W];
                if (whole_rows && left >= W) {
#pragma unroll
                    for (int i = 0; i < W; ++i) raw[i] = c[i * p.ldc];
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) raw[i] = m < p.M && i < left ? c[i * p.ldc] : static_cast<unsigned short>(0);
                }
#pragma unroll
                for (int i = 0; i < W; ++i)
                    c_next[i] = p.c_fmt == 2 ? __uint_as_float(static_cast<uint32_t>(raw[i]) << 16) : __half2float(__ushort_as_half(raw[i]));
            }
        };
        if (has_c && !sends && kSplit != 4) prefetch_c(u);
        if (kAhead && has_c && !sends && cols > 0 && kSplit != 4) load_c(0);

        // W columns from column j * W of this warp group on: the whole warp, `ok` in every lane
        auto finish = [&](int j, uint32_t (&r)[W]) {
            if constexpr (kSplit == 2) {
                if (sends || receives) exchange(r);
                if (sends || !ok) return;
            }
            const int n = u.n0 + col0 + j * W, left = cols - j * W;
            if (has_c) {
                if (!kAhead) load_c(j);
#pragma unroll
                for (int i = 0; i < W; ++i) r[i] = __float_as_uint(fmaf(alpha, __uint_as_float(r[i]), beta * c_next[i]));
                if (kAhead && (j + 1) * W < cols) load_c(j + 1);
            } else {
#pragma unroll
                for (int i = 0; i < W; i += 2) {
                    if constexpr (kF32) {
                        r[i] = __float_as_uint(alpha * __uint_as_float(r[i]));
                        r[i + 1] = __float_as_uint(alpha * __uint_as_float(r[i + 1]));
                    } else {
                        const float2 x = __fmul2_rn(make_float2(alpha, alpha), make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
                        r[i] = __float_as_uint(x.x);
                        r[i + 1] = __float_as_uint(x.y);
                    }
                }
            }
            const long long at = (kPerGroup ? u.group * p.stride_d : 0) + m + n * p.ldd;
            if (d_fmt == 0) {
                float* d = static_cast<float*>(p.D) + at;
                if (whole_rows && left >= W) {
#pragma unroll
                    for (int i = 0; i < W; ++i, d += p.ldd) *d = __uint_as_float(r[i]);
                } else if (m < p.M) {
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (i < left) d[i * p.ldd] = __uint_as_float(r[i]);
                }
                return;
            }
            if constexpr (!kF32) {
                uint32_t v[W / 2];  // columns 2 i and 2 i + 1, rounded
                if (d_fmt == 2) {
#pragma unroll
                    for (int i = 0; i < W; i += 2) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                        v[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < W; i += 2) {
                        const __half2 h = __floats2half2_rn(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                        v[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                }
                unsigned short* d = static_cast<unsigned short*>(p.D) + at;
                if (whole_rows && left >= W && p.d_pairs) {
                    // the even lane stores rows m, m + 1 of the first column of two, the odd lane m - 1, m of the second
                    const int odd = lane & 1;
                    const uint32_t pick = odd ? 0x3276u : 0x5410u;
                    d += odd * (p.ldd - 1);
#pragma unroll
                    for (int i = 0; i < W; i += 2) {
                        const uint32_t x = __shfl_xor_sync(0xffffffffu, v[i / 2], 1);
                        *reinterpret_cast<uint32_t*>(d) = __byte_perm(v[i / 2], x, pick);
                        d += 2 * p.ldd;
                    }
                } else if (m < p.M) {
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (i < left) d[i * p.ldd] = static_cast<unsigned short>(v[i / 2] >> (16 * (i & 1)));
                }
            }
        };

        // four CTAs: this thread's row of the warp group's 32 columns goes to two of them; the first warp group adds
        // and stores this CTA's own columns
        auto deal = [&](const float (&sum)[E::COLS]) {
            constexpr int kShare = 2 * E::COLS / kSplit;  // columns of one CTA
            ok = ok && mbar_wait_cluster(split.empty_bar, (split_count & 1u) ^ 1u, wc, kWaitPartial);  // room everywhere
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            const uint32_t at = split.recv_addr + (split.role * 128 + et) * kShare * 4;
#pragma unroll
            for (int q = 0; q < E::COLS / kShare; ++q) {
                const uint32_t rank = wg * (E::COLS / kShare) + q, to = mapa_shared(at, rank), bar = mapa_shared(split.full_bar, rank);
#pragma unroll
                for (int i = 0; i < kShare; i += 4) {
                    uint32_t v[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = __float_as_uint(sum[q * kShare + i + x]);
                    st_async_cluster(to + i * 4, v, bar);
                }
            }
            if (wg == 0) {
                if (et == 0) mbar_arrive_expect_tx(split.full_bar, kSplit * 128 * kShare * 4);
                ok = mbar_wait_cluster(split.full_bar, split_count & 1u, wc, kWaitPartial);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                float v[kShare] = {};
#pragma unroll
                for (int src = 0; src < kSplit; ++src) {
                    const float4* in = reinterpret_cast<const float4*>(split.recv + (src * 128 + et) * kShare);
#pragma unroll
                    for (int i = 0; i < kShare / 4; ++i) {
                        const float4 x = in[i];
                        v[4 * i] += x.x;
                        v[4 * i + 1] += x.y;
                        v[4 * i + 2] += x.z;
                        v[4 * i + 3] += x.w;
                    }
                }
                __syncwarp();
                if (lane < kSplit) mbar_arrive_cluster(split.empty_bar, lane);
                const int n = u.n0 + split.role * kShare, left = u.cols - split.role * kShare;
                const long long c_at = (kPerGroup ? u.group * p.stride_c : 0) + m + n * p.ldc;
                const long long d_at = (kPerGroup ? u.group * p.stride_d : 0) + m + n * p.ldd;
#pragma unroll
                for (int i = 0; i < kShare; ++i) {
                    if (m >= p.M || i >= left) continue;
                    float x = alpha * v[i];
                    if (has_c) {
                        const long long e = c_at + i * p.ldc;
                        const float c = p.c_fmt == 2   ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.C)[e])
                                        : p.c_fmt == 1 ? __half2float(static_cast<const __half*>(p.C)[e])
                                                       : static_cast<const float*>(p.C)[e];
                        x = fmaf(beta, c, x);
                    }
                    const long long e = d_at + i * p.ldd;
                    if (d_fmt == 2) static_cast<__nv_bfloat16*>(p.D)[e] = __float2bfloat16_rn(x);
                    else if (d_fmt == 1) static_cast<__half*>(p.D)[e] = __float2half_rn(x);
                    else static_cast<float*>(p.D)[e] = x;
                }
            }
            ++split_count;
        };

        if constexpr (kPromoteKb > 0) {
            float sum[E::COLS];
#pragma unroll
            for (int i = 0; i < E::COLS; ++i) sum[i] = 0.0f;
            for (int kb = 0; ok && kb < u.kb; kb += (kPromoteKb > 0 ? kPromoteKb : 1), ++acc_count) {
                const uint32_t acc = acc_count % kAccs;
                wait_acc(acc);
                if (!ok) break;
#pragma unroll
                for (int q = 0; q < E::COLS / W; ++q) {
                    if (q * W < cols) {
                        uint32_t r[W];
                        tmem_ld_32x32b_x32(tmem_base + lane_base + acc * kBN + col0 + q * W, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < W; ++i) sum[q * W + i] += __uint_as_float(r[i]);
                    }
                }
                release(acc);
            }
            if constexpr (kSplit == 4) deal(sum);
#pragma unroll
            for (int q = 0; q < (kSplit == 4 ? 0 : E::COLS / W); ++q) {
                if (ok && q * W < cols) {
                    uint32_t r[W];
#pragma unroll
                    for (int i = 0; i < W; ++i) r[i] = __float_as_uint(sum[q * W + i]);
                    finish(q, r);
                }
            }
        } else if constexpr (kDrain) {
            uint32_t r[E::COLS / W][W];
            const uint32_t acc = acc_count % kAccs;
            wait_acc(acc);
            if (!ok) break;
#pragma unroll
            for (int q = 0; q < E::COLS / W; ++q)
                if (q * W < cols) tmem_ld_32x32b_x32(tmem_base + lane_base + acc * kBN + col0 + q * W, r[q]);
            tmem_wait_ld();
            release(acc);
            ++acc_count;
            // the issuer waits for each of the further ones to be read: its sum stays in the registers
            for (int kb = p.whole_kb; kLong && kb < u.kb; kb += p.whole_kb, ++acc_count) {
                const uint32_t acc = acc_count % kAccs;
                wait_acc(acc);
                if (!ok) break;
#pragma unroll
                for (int q = 0; q < E::COLS; q += 16) {
                    if (q < cols) {
                        uint32_t x[16];
                        tmem_ld_32x32b_x16(tmem_base + lane_base + acc * kBN + col0 + q, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) r[q / W][q % W + i] = __float_as_uint(__uint_as_float(r[q / W][q % W + i]) + __uint_as_float(x[i]));
                    }
                }
                release(acc);
            }
            if (!ok) break;
#pragma unroll
            for (int q = 0; q < E::COLS / W; ++q)
                if (ok && q * W < cols) finish(q, r[q]);
        } else {
            const bool empty = u.kb == 0;
            const uint32_t acc = acc_count % kAccs;
            if (!empty && !longer) wait_acc(acc);
            if (!ok) break;
            for (int j = 0; ok && j * W < cols; ++j) {
                uint32_t r[W];
                if (!empty) {
                    tmem_ld_32x32b_x32(tmem_base + lane_base + acc * kBN + col0 + j * W, r);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) r[i] = 0u;
                }
                finish(j, r);
            }
            if (!empty) {
                release(acc);
                ++acc_count;
            }
        }
        if (!ok) break;
    }
}

}  // namespace b200
