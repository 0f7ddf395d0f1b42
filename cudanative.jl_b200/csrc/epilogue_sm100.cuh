// Epilogue shared by the grouped and the 4-bit products: D = alpha * acc + beta * C from accumulators in
// tensor memory, by two groups of four warps, each with one half of a tile's columns.
//
// Why two groups: with short inner dimensions (a group's tokens, four-bit operands) a tile's main loop
// takes as long as reading its accumulator, and one group of warps converts 128 x 256 values in about
// the 4 000 cycles of eight k-blocks.
//
// kPromote: the tensor core adds into its accumulator without rounding to nearest; every step drops what
// lies below the last place, which pulls sums towards zero in proportion to the number of steps (measured
// on K = 4096: 4e-6 of the result, 2e-5 for K = 16384; on K = 256 3e-7).  For a binary32 D that is more
// than the result's own precision, so the MMA issuer starts a new accumulator every PROMOTE_KB k-blocks
// and the warps add it, rounding to nearest, to a running sum in their registers while the next one is
// being filled.  A 16-bit D rounds at 2^-9 or 2^-12 and takes the whole sum from one accumulator.
//
// A chunk of W columns is staged in shared memory and stored by one bulk copy; a chunk that may not be
// written whole (a group's ragged end, rows that are no multiple of 16 bytes) is stored from registers.
// C comes by bulk copies C_AHEAD chunks ahead where its rows allow it (c_tma), else from registers too.
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
    int c_tma, d_tma;                        // may be moved by bulk copies
};

// A tile of work: this CTA's first row, the tile's first column, the columns that exist; the inner dimension
// from k0 on, of which this CTA takes k-blocks (of 64 or 256) kb0 .. kb0 + kb - 1.
struct Unit {
    int group, m0, n0, cols, k0, k_len, kb0, kb;
};

// With few tiles the two CTAs of a cluster take half of a tile's inner dimension each: CTA 1 sends its sums
// into CTA 0's shared memory, CTA 0 adds them to its own (always in this order) and stores.
struct SplitParams {
    int role = -1;       // -1: whole tiles, 0: receives and stores, 1: sends
    const float* recv;   // [columns][128]
    uint32_t recv_addr;
    uint32_t full_bar, empty_bar;
};

// kW: 16 columns of up to 4 bytes, or 32 columns of 2 bytes (16-bit D without bulk loads of C).
template <int kBN, int kW, bool kBulkC, int kBufs = 3>
struct EpilogueCfg {
    static constexpr int COLS = kBN >= 64 ? kBN / 2 : kBN;  // per warp group; the second is idle below 64
    static constexpr int W = kW;
    static constexpr int BUFS = kBufs;
    static constexpr int BUF_BYTES = 8192;
    static constexpr int C_AHEAD = BUFS - 1;
    static constexpr bool BULK_C = kBulkC;
    static constexpr int BYTES = 2 * BUFS * BUF_BYTES;
    static_assert(COLS % kW == 0 && (kW == 16 || (kW == 32 && !kBulkC)), "chunks");
};

__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_32x32b_x16(taddr, r); }
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32b_x32(taddr, r); }

constexpr int kDrain = 1 << 30;  // kPromoteKb: one accumulator per tile, moved to registers before the rest

// Runs in warps 4 .. 11 (`wg` 0 or 1).  Barriers: tmem_full / tmem_empty [kAccs] at the given addresses,
// 8 bytes apart; cfull [BUFS] of this warp group.
template <class E, int kBN, int kAccs, int kCtas, bool kF32, int kPromoteKb, bool kPerGroup, bool kSplit, class Decode>
__device__ __forceinline__ void run_epilogue(const EpilogueParams& p, const CUtensorMap* tmC, const CUtensorMap* tmD, int wg, uint32_t tmem_base,
                                             uint32_t epi_base, uint8_t* epi_gen, uint32_t tmem_full, uint32_t tmem_empty, uint32_t cfull,
                                             const WaitCtx& wc, int unit_first, int unit_stride, int num_units, const SplitParams& split, Decode decode) {
    constexpr int W = E::W, BUFS = E::BUFS;
    const int et = static_cast<int>(threadIdx.x & 127);
    const int lane = static_cast<int>(threadIdx.x & 31);
    const uint32_t lane_base = static_cast<uint32_t>(((threadIdx.x >> 5) & 3) * 32) << 16;
    const bool elected = et == 0;
    const uint32_t bar = 1 + 3 * wg;  // named barriers of this warp group
    const bool has_c = p.beta != 0.0f;
    const bool c_bulk = E::BULK_C && has_c && p.c_tma;
    const float alpha = p.alpha, beta = p.beta;
    const int d_fmt = kF32 ? 0 : p.d_fmt;
    const bool c_half = p.c_fmt != 0, d_half = d_fmt != 0;
    const uint32_t c_chunk_bytes = 128 * W * (c_half ? 2 : 4);
    const bool two_phase = c_bulk && (c_half != d_half);
    const uint64_t stream_policy = l2_policy_evict_first();
    auto own_cols = [&](const Unit& u) { return min(E::COLS, max(0, u.cols - wg * E::COLS)); };

    // the chunks of C this warp group will need, asked for C_AHEAD chunks ahead
    uint32_t g = 0, asked = 0;
    int pf_unit = unit_first, pf_j = 0, pf_cols = 0;
    Unit pf = {};
    auto fetch_c = [&]() {
        if constexpr (E::BULK_C) {
            while (pf_j * W >= pf_cols) {  // next unit with columns for this warp group
                if (pf_unit >= num_units) return;
                pf = decode(pf_unit);
                pf_unit += unit_stride;
                pf_cols = own_cols(pf);
                pf_j = 0;
            }
            const uint32_t b = asked % BUFS;
            const int y = pf.n0 + wg * E::COLS + pf_j * W;
            mbar_arrive_expect_tx(cfull + 8 * b, c_chunk_bytes);
            tma_load_3d_hint(epi_base + b * E::BUF_BYTES, tmC, pf.m0, y, pf.group, cfull + 8 * b, stream_policy);
            ++asked;
            ++pf_j;
        }
    };
    if (c_bulk && elected)
        for (int i = 0; i < E::C_AHEAD; ++i) fetch_c();

    uint32_t acc_count = 0, split_count = 0;
    bool fail = false, ok = true;
    const bool sends = kSplit && split.role == 1, receives = kSplit && split.role == 0;
    const uint32_t remote = kSplit ? mapa_shared(split.recv_addr, 0) : 0u;
    // room in the receiver's buffer, or the sender's sums in it
    auto split_begin = [&]() {
        if (sends) ok = ok && mbar_wait_cluster(split.empty_bar, (split_count & 1u) ^ 1u, wc, kWaitPartial);
        if (receives) ok = ok && mbar_wait_cluster(split.full_bar, split_count & 1u, wc, kWaitPartial);
        ok = __all_sync(0xffffffffu, ok);
    };
    auto split_chunk = [&](int j, uint32_t (&r)[W]) {
        if (!ok) return;
        if (sends) {
#pragma unroll
            for (int i = 0; i < W; ++i) st_cluster_u32(remote + ((j * W + i) * 128 + et) * 4, r[i]);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + split.recv[(j * W + i) * 128 + et]);
        }
    };
    auto split_end = [&]() {
        __syncwarp();
        if (lane == 0 && sends) mbar_arrive_cluster(split.full_bar, 0);
        if (lane == 0 && receives) mbar_arrive_cluster(split.empty_bar, 1);
        ++split_count;
    };
    for (int unit = unit_first; unit < num_units; unit += unit_stride) {
        const Unit u = decode(unit);
        const int cols = own_cols(u);
        const int col0 = wg * E::COLS;
        const int m = u.m0 + et;

        // alpha * r + beta * C, into the staging buffer or to D; returns true to go on
        auto finish = [&](int j, uint32_t (&r)[W]) {
            const uint32_t buf = g % BUFS;
            float* col = reinterpret_cast<float*>(epi_gen + buf * E::BUF_BYTES) + et;
            __half* colh = reinterpret_cast<__half*>(epi_gen + buf * E::BUF_BYTES) + et;
            __nv_bfloat16* colb = reinterpret_cast<__nv_bfloat16*>(colh);
            const int n = u.n0 + col0 + j * W;
            // D_e's own right edge is clipped by its tensor map; a group's border inside D is not
            const bool bulk = p.d_tma && (kPerGroup || (j + 1) * W <= cols);
            if (ok) {
                if (c_bulk) {
                    if (p.c_fmt == 2) {
#pragma unroll
                        for (int i = 0; i < W; ++i) r[i] = __float_as_uint(fmaf(alpha, __uint_as_float(r[i]), beta * __bfloat162float(colb[i * 128])));
                    } else if (c_half) {
#pragma unroll
                        for (int i = 0; i < W; ++i) r[i] = __float_as_uint(fmaf(alpha, __uint_as_float(r[i]), beta * __half2float(colh[i * 128])));
                    } else {
#pragma unroll
                        for (int i = 0; i < W; ++i) r[i] = __float_as_uint(fmaf(alpha, __uint_as_float(r[i]), beta * col[i * 128]));
                    }
                } else if (has_c) {
                    const long long at = (kPerGroup ? u.group * p.stride_c : 0) + m + n * p.ldc;
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        float c = 0.0f;
                        if (m < p.M && j * W + i < cols) {
                            const long long e = at + i * p.ldc;
                            c = p.c_fmt == 2 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.C)[e])
                                : c_half     ? __half2float(static_cast<const __half*>(p.C)[e])
                                             : static_cast<const float*>(p.C)[e];
                        }
                        r[i] = __float_as_uint(fmaf(alpha, __uint_as_float(r[i]), beta * c));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) r[i] = __float_as_uint(alpha * __uint_as_float(r[i]));
                }
            }
            if (two_phase) named_bar_sync(bar + 2, 128);
            if (ok && bulk) {
                if (d_fmt == 2) {
#pragma unroll
                    for (int i = 0; i < W; ++i) colb[i * 128] = __float2bfloat16_rn(__uint_as_float(r[i]));
                } else if (d_half) {
#pragma unroll
                    for (int i = 0; i < W; ++i) colh[i * 128] = __float2half_rn(__uint_as_float(r[i]));
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) col[i * 128] = __uint_as_float(r[i]);
                }
                fence_proxy_async_smem();
            } else if (ok && m < p.M) {
                const long long at = (kPerGroup ? u.group * p.stride_d : 0) + m + n * p.ldd;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    if (j * W + i < cols) {
                        const long long e = at + i * p.ldd;
                        if (d_fmt == 2) static_cast<__nv_bfloat16*>(p.D)[e] = __float2bfloat16_rn(__uint_as_float(r[i]));
                        else if (d_half) static_cast<__half*>(p.D)[e] = __float2half_rn(__uint_as_float(r[i]));
                        else static_cast<float*>(p.D)[e] = __uint_as_float(r[i]);
                    }
                }
            }
            fail = named_bar_or(bar + 1, 128, !ok);
            if (fail) return false;
            if (elected) {
                if (c_bulk) {
                    tma_store_wait_read<0>();  // the store before this one has let go of the buffer that is refilled
                    fetch_c();
                }
                if (bulk && u.m0 < p.M) {
                    if constexpr (kPerGroup) tma_store_3d_hint(tmD, u.m0, n, u.group, epi_base + buf * E::BUF_BYTES, stream_policy);
                    else tma_store_2d(tmD, u.m0, n, epi_base + buf * E::BUF_BYTES);
                }
                tma_store_commit();  // without a store too: the count of groups is the count of buffers
            }
            ++g;
            return true;
        };
        // before a chunk's buffer is touched: C has landed in it, or the store that last read it is done
        auto buffer_ready = [&]() {
            if (c_bulk) {
                ok = ok && mbar_wait(cfull + 8 * (g % BUFS), (g / BUFS) & 1u, wc, kWaitCTile);
            } else {
                if (elected) tma_store_wait_read<BUFS - 1>();
                named_bar_sync(bar, 128);
            }
            ok = __all_sync(0xffffffffu, ok);  // tcgen05.ld is warp-collective
        };
        auto release = [&](uint32_t acc) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kCtas == 2) mbar_arrive_cluster(tmem_empty + 8 * acc, 0);
                else mbar_arrive(tmem_empty + 8 * acc);
            }
        };

        if constexpr (kPromoteKb >= kDrain) {
            // one accumulator in tensor memory: read it out at once and let the next tile begin
            uint32_t r[E::COLS / W][W];
            const uint32_t acc = acc_count % kAccs;
            ok = ok && mbar_wait(tmem_full + 8 * acc, (acc_count / kAccs) & 1u, wc, kWaitTmemFull);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after_sync();
            if (ok) {
#pragma unroll
                for (int q = 0; q < E::COLS / W; ++q)
                    if (q * W < cols) tmem_ld_cols(tmem_base + lane_base + acc * kBN + col0 + q * W, r[q]);
                tmem_wait_ld();
            }
            release(acc);
            ++acc_count;
#pragma unroll
            for (int q = 0; q < E::COLS / W; ++q) {
                if (!fail && q * W < cols) {
                    buffer_ready();
                    finish(q, r[q]);
                }
            }
            if (fail) break;
        } else if constexpr (kPromoteKb > 0) {
            float sum[E::COLS];
#pragma unroll
            for (int i = 0; i < E::COLS; ++i) sum[i] = 0.0f;
            for (int kb = 0; kb < u.kb; kb += kPromoteKb, ++acc_count) {
                const uint32_t acc = acc_count % kAccs;
                ok = ok && mbar_wait(tmem_full + 8 * acc, (acc_count / kAccs) & 1u, wc, kWaitTmemFull);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after_sync();
                if (ok) {
#pragma unroll
                    for (int q = 0; q < E::COLS / W; ++q) {
                        if (q * W < cols) {
                            uint32_t r[W];
                            tmem_ld_cols(tmem_base + lane_base + acc * kBN + col0 + q * W, r);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < W; ++i) sum[q * W + i] += __uint_as_float(r[i]);
                        }
                    }
                }
                release(acc);
            }
            if (kSplit && (sends || receives) && cols > 0) split_begin();
#pragma unroll
            for (int q = 0; q < E::COLS / W; ++q) {
                if (!fail && q * W < cols) {
                    uint32_t r[W];
                    if (!sends) buffer_ready();
#pragma unroll
                    for (int i = 0; i < W; ++i) r[i] = __float_as_uint(sum[q * W + i]);
                    if (kSplit && (sends || receives)) split_chunk(q, r);
                    if (!sends) finish(q, r);
                }
            }
            if (kSplit && (sends || receives) && cols > 0) split_end();
            if (fail || (sends && !ok)) break;
        } else {
            const bool empty = u.kb == 0;
            const uint32_t acc = acc_count % kAccs;
            if (!empty) ok = ok && mbar_wait(tmem_full + 8 * acc, (acc_count / kAccs) & 1u, wc, kWaitTmemFull);
            tc_fence_after_sync();
            if (kSplit && (sends || receives) && cols > 0) split_begin();
            for (int j = 0; j * W < cols; ++j) {
                if (sends) ok = __all_sync(0xffffffffu, ok);
                else buffer_ready();
                uint32_t r[W];
                if (ok && !empty) {
                    tmem_ld_cols(tmem_base + lane_base + acc * kBN + col0 + j * W, r);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) r[i] = 0u;
                }
                if (kSplit && (sends || receives)) split_chunk(j, r);
                if (!sends && !finish(j, r)) break;
            }
            if (kSplit && (sends || receives) && cols > 0) split_end();
            if (fail || (sends && !ok)) break;
            if (!empty) {
                release(acc);
                ++acc_count;
            }
        }
    }
    if (elected) tma_store_wait_all<0>();
}

}  // namespace b200
