// Product of two microscaled 4-bit matrices for sm_100a, plain or grouped with ragged columns:
//
//   D[:, s_e] = alpha * A_e^T * B[:, s_e] + beta * C[:, s_e]
//
// A_e is K x M and B is K x N, elements and scales as mxfp4.cu lays them out; without offsets there is one
// group of all columns.
//
// The pipeline is that of gemm_grouped.cuh with 256 values of k (128 bytes of elements) per stage, four
// tcgen05.mma.kind::mxf4.block_scale of K = 64 each, and the stage's scales: one 512-byte tile per 128 rows
// and 128 values of k, brought by bulk copies of its own.  The products read scales from tensor memory, the
// same 32 lanes repeated in each warp's quarter: four more warps (12 - 15) carry them there, one quarter each,
// a set of columns per stage.  (tcgen05.cp does the same from the MMA issuer's thread, but holds up the
// products behind it by about 80 cycles a tile, six tiles to 512 cycles of products: 8192^3 took 370 us,
// 437 us with the copies issued one stage ahead, and 266 us with the four warps.)
//
// A tile's scales always come from whole tiles of 128 columns, counted from the group's first column, as
// they were quantised.  A tile of 32 columns may begin at row 32, 64 or 96 of one: the warps that carry its
// scales put those rows into the first column, since an odd column is no legal scale address.  A tile of 192
// begins at row 0 or 64, which is column 0 or 2.
//
// How long a sum one accumulator may take: the tensor core truncates when it adds, and though 4-bit products have few bits, sums of
// one sign whose scales differ lose some with every instruction (scales within 2^+-4, one accumulator: 8e-7 of the
// result at K = 8192, 1.4e-5 at 65536, 7e-5 at 262144).  A binary32 D takes 8192 products from one accumulator, a 16-bit D
// 65536; a longer K has a kernel of its own (kLong) that adds several with rounding to nearest.
//
// What bounds it: 4-bit products run at four times the rate of 16-bit ones, with the same bytes per cycle.
// For few columns (a token, a decode step) the elements of A, 17/32 byte per value, are the floor.
#pragma once

#include <type_traits>

#include "gemm_grouped.cuh"
#include "mx_scale_rows.h"

namespace b200 {

struct MxGemmParams {
    int N, K;
    int groups;
    Raster raster;
    const int* offsets;  // nullptr: one group, all columns
    int a_per_group;
    int a_tile_rows;     // rows of scale tiles of one A_e
    EpilogueParams e;
    int* status;
    unsigned long long wait_budget_ns;
};

template <int kBN, int kCtas, bool kSplit>
struct MxCfg {
    static constexpr int THREADS = 512;
    static constexpr int BM = 128;
    static constexpr int BK = 256;  // values of k per stage
    static constexpr int BN_LOCAL = kBN / kCtas;
    static constexpr int A_BYTES = BM * BK / 2;
    static constexpr int B_BYTES = BN_LOCAL * BK / 2;
    static constexpr int B_TILES = (kBN + 127) / 128;  // scale tiles that a tile of columns touches at most
    static constexpr int SF_BYTES = 1024 * (1 + B_TILES);
    static constexpr int STAGE_BYTES = (A_BYTES + B_BYTES + SF_BYTES + 1023) / 1024 * 1024;
    static constexpr int BBOX = BN_LOCAL < 128 ? BN_LOCAL : 128;
    static constexpr int BBOX_BYTES = BBOX * BK / 2;
    static constexpr int GRANULE = kCtas == 2 ? 32 : 16;
    using Epi = EpilogueCfg<kBN>;
    static constexpr int TABLE_BYTES = 3 * (kMaxGroups + 4) * 4;
    static constexpr int BAR_BYTES = 512;
    static constexpr int SCAN_AT = 384;  // among them, behind the barriers: scratch of the groups' scan, a sum per warp
    static constexpr int RECV_BYTES = kSplit ? 128 * kSplitRow * 4 : 0;
    static constexpr int BUDGET = 227 * 1024 - 1024 - BAR_BYTES - TABLE_BYTES - RECV_BYTES;
    static constexpr int ACCS = kBN <= 192 ? 2 : 1;
    static constexpr int SCALE_COLS = 8 * (1 + B_TILES);  // per set: 2 x 4 for A, 2 x 4 per scale tile for B
    static constexpr int SCALE_AT = ACCS * kBN;
    static constexpr int MOST = (512 - SCALE_AT) / SCALE_COLS < 8 ? (512 - SCALE_AT) / SCALE_COLS : 8;  // a set of scales per stage
    static constexpr int STAGES = BUDGET / STAGE_BYTES > MOST ? MOST : BUDGET / STAGE_BYTES;
    static constexpr int USED_COLS = SCALE_AT + STAGES * SCALE_COLS;
    static constexpr int TMEM_COLS = USED_COLS <= 128 ? 128 : USED_COLS <= 256 ? 256 : 512;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + RECV_BYTES + TABLE_BYTES + BAR_BYTES + 1024;
    static constexpr int NBARS = 3 * STAGES + 2 + 2 * ACCS;
    static_assert(!kSplit || (kCtas == 1 && kBN <= 32), "split inner dimension: one-CTA tiles, one warp group");
    static_assert(USED_COLS <= 512, "tensor memory");
    static_assert(STAGES >= 3 && SMEM_BYTES <= 227 * 1024, "shared memory");
    static_assert(8 * NBARS + 8 <= SCAN_AT && SCAN_AT + THREADS / 32 * 8 <= BAR_BYTES, "barriers, scratch");
    static_assert(kBN == 32 || kBN == 128 || kBN == 192 || kBN == 256, "a tile of columns begins on a multiple of 32 inside its scale tile");
};

// k-blocks that one accumulator sums at most
__host__ __device__ constexpr int mx_whole_kb(int d_fmt) { return d_fmt == 0 ? 32 : 256; }

template <int kBN, int kCtas, bool kSplit, bool kLong>
__global__ void __launch_bounds__(512, 1)
gemm_mxfp4_tcgen05(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const MxGemmParams p) {
    using Cfg = MxCfg<kBN, kCtas, kSplit>;
    using Epi = typename Cfg::Epi;
    constexpr int STAGES = Cfg::STAGES, ACCS = Cfg::ACCS;
    constexpr bool kPair = (kCtas == 2);

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    constexpr int kRecvAt = STAGES * Cfg::STAGE_BYTES;
    constexpr int kTableAt = kRecvAt + Cfg::RECV_BYTES;
    const uint32_t bar_base = smem_base + kTableAt + Cfg::TABLE_BYTES;
    int* off = reinterpret_cast<int*>(smem_gen + kTableAt);
    int* first = off + kMaxGroups + 4;
    int* first128 = kBN == 128 ? first : first + kMaxGroups + 4;  // scale tiles before each group
    uint8_t* bar_gen = smem_gen + kTableAt + Cfg::TABLE_BYTES;

    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto scales_full_bar = [&](int s) { return bar_base + 8u * (2 * STAGES + s); };   // in this CTA's shared memory
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (3 * STAGES + a); };
    auto tmem_empty_bar = [&](int a) { return bar_base + 8u * (3 * STAGES + ACCS + a); };
    auto split_bar = [&](int i) { return bar_base + 8u * (3 * STAGES + 2 * ACCS + i); };  // partial sums: full, empty
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bar_gen + 8 * Cfg::NBARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_gen + 8 * Cfg::NBARS + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = kPair ? cluster_cta_rank() : 0u;
    int unit_stride = kPair ? (gridDim.x >> 1) : gridDim.x;
    int unit_first = kPair ? (blockIdx.x >> 1) : blockIdx.x;
    WaitCtx wc{abort_flag, p.status, p.wait_budget_ns};

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1 + 4 * kCtas);  // the leader's producer; the warps that carry scales
            mbar_init(empty_bar(s), 1);
            mbar_init(scales_full_bar(s), 1);
        }
        for (int a = 0; a < ACCS; ++a) {
            mbar_init(tmem_full_bar(a), 1);
            mbar_init(tmem_empty_bar(a), 8 * kCtas);
        }
        mbar_init(split_bar(0), 1);  // the receiver's arrive; it expects the sender's bytes
        mbar_init(split_bar(1), 4);  // the receiver's four warps
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        tma_prefetch_desc(&tmSA);
        tma_prefetch_desc(&tmSB);
    }
    if (warp == 2) tmem_alloc<kCtas>(smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::TMEM_COLS);
    tc_fence_before_sync();
    __syncthreads();
    if constexpr (kPair || kSplit) cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch_dependents();
    griddep_wait();

    const bool offsets_ok = load_groups<true, Cfg::THREADS>(p.offsets, p.groups, p.N, kBN, off, first, reinterpret_cast<unsigned long long*>(bar_gen + Cfg::SCAN_AT),
                                                            kBN == 128 ? nullptr : first128);
    if (!offsets_ok && threadIdx.x == 0) report_bad_offsets(p.status, p.groups);
    const int num_units = offsets_ok ? first[p.groups] * p.raster.rows.d : 0;

    // Split the inner dimension when that shortens the longest CTA's work (counted in whole tiles).
    SplitParams split;
    const int kb_all = (p.K + Cfg::BK - 1) / Cfg::BK;
    if constexpr (kSplit) {
        const int ctas = gridDim.x;
        const int whole = (num_units + ctas - 1) / ctas, halves = (num_units + ctas / 2 - 1) / (ctas / 2);
        if (kb_all >= 4 && halves < 2 * whole) {
            split.role = static_cast<int>(cluster_cta_rank());
            unit_first = blockIdx.x >> 1;
            unit_stride = ctas >> 1;
        }
        split.recv = reinterpret_cast<const float*>(smem_gen + kRecvAt);
        split.recv_addr = smem_base + kRecvAt;
        split.full_bar = split_bar(0);
        split.empty_bar = split_bar(1);
    }
    // this CTA's k-blocks of every tile
    const int kb_half = (kb_all + 1) / 2;
    const int kb_first = kSplit && split.role == 1 ? kb_half : 0;
    const int kb_total = !kSplit || split.role < 0 ? kb_all : split.role ? kb_all - kb_half : kb_half;

    auto decode = [&](int unit) {
        Unit u;
        u.group = find_group(first, p.groups, unit / p.raster.rows);
        const int2 tile = place_tile(p.raster, unit - first[u.group] * p.raster.rows.d, first[u.group + 1] - first[u.group]);
        u.m0 = tile.x * (Cfg::BM * kCtas) + static_cast<int>(cta_rank) * Cfg::BM;
        u.n0 = off[u.group] + tile.y * kBN;
        u.cols = min(kBN, off[u.group + 1] - u.n0);
        u.k0 = 0;
        u.k_len = p.K;
        u.kb0 = kb_first;
        u.kb = kb_total;
        return u;
    };
    auto inst_n = [&](const Unit& u) { return (u.cols + Cfg::GRANULE - 1) / Cfg::GRANULE * Cfg::GRANULE; };
    // of a tile's first column among the 128 of its scale tile
    auto scale_shift = [&](const Unit& u) { return (u.n0 - off[u.group]) & 127; };

    // registers: 4 x 128 a thread at launch = 2 x 56 + 2 x 200; the epilogue holds half a tile row in them
    if (warp < 4) {
        regs_dec<56>();
        if (warp == 0) {
            // ------------------------------------------------------------------ TMA producer
            if (lane == 0) {
                int s = 0;
                uint32_t ph = 0;
                bool ok = true;
                const uint64_t once = l2_policy_evict_first();
                for (int unit = unit_first; ok && unit < num_units; unit += unit_stride) {
                    const Unit u = decode(unit);
                    const int ninst = inst_n(u);
                    const int nb0 = u.n0 + static_cast<int>(cta_rank) * (ninst / kCtas);
                    const int boxes = (ninst / kCtas + Cfg::BBOX - 1) / Cfg::BBOX;
                    const bool a_once = first[u.group + 1] - first[u.group] == 1;
                    const int z = u.group * p.a_per_group;
                    const uint32_t bytes = Cfg::A_BYTES + boxes * Cfg::BBOX_BYTES;
                    for (int kb = 0; kb < u.kb; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0)) {
                        ok = mbar_wait(empty_bar(s), ph ^ 1u, wc, kWaitEmptyStage);
                        if (!ok) break;
                        const uint32_t at_a = smem_base + s * Cfg::STAGE_BYTES;
                        const uint32_t at_b = at_a + Cfg::A_BYTES;
                        uint32_t fb = full_bar(s);
                        if constexpr (kPair) fb = mapa_shared(fb, 0);
                        if (cta_rank == 0) mbar_arrive_expect_tx(full_bar(s), kCtas * bytes);
                        if constexpr (kPair) tma_load_3d_pair(at_a, &tmA, (kb_first + kb) * 128, u.m0, z, fb);
                        else if (a_once) tma_load_3d_hint(at_a, &tmA, (kb_first + kb) * 128, u.m0, z, fb, once);
                        else tma_load_3d(at_a, &tmA, (kb_first + kb) * 128, u.m0, z, fb);
                        auto load = [&](uint32_t dst, const CUtensorMap* tm, int x, int y) {
                            if constexpr (kPair) tma_load_2d_pair(dst, tm, x, y, fb);
                            else tma_load_2d(dst, tm, x, y, fb);
                        };
                        for (int i = 0; i < boxes; ++i) load(at_b + i * Cfg::BBOX_BYTES, &tmB, (kb_first + kb) * 128, nb0 + i * Cfg::BBOX);
                    }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------------------------ MMA issuer
            if (cta_rank == 0) {
                const uint32_t lead = elect_lane();
                const uint64_t da0 = make_smem_desc(smem_base, 16, 1024, kSwizzle128B);
                const uint64_t db0 = make_smem_desc(smem_base + Cfg::A_BYTES, 16, 1024, kSwizzle128B);
                int s = 0;
                uint32_t ph = 0, ucount = 0;
                bool ok = true, ready = false;
                for (int unit = unit_first; ok && unit < num_units; unit += unit_stride) {
                    const Unit u = decode(unit);
                    // 192 columns begin at row 0 or 64 of their scale tile: two columns of 32 rows further
                    const uint32_t shift = kBN == 192 ? __shfl_sync(0xffffffffu, static_cast<uint32_t>(scale_shift(u)) / 32, 0) : 0u;
                    const uint32_t idesc0 = make_idesc_mxf4(Cfg::BM * kCtas, __shfl_sync(0xffffffffu, inst_n(u), 0), 0);
                    uint32_t acc, d_tmem;
                    auto begin = [&] {
                        acc = ucount % ACCS;
                        d_tmem = tmem_base + acc * kBN;
                        ok = __all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(acc), ((ucount / ACCS) & 1u) ^ 1u, wc, kWaitTmemEmpty));
                    };
                    auto end = [&] {
                        if (lead) {
                            if constexpr (kPair) umma_commit_pair(tmem_full_bar(acc));
                            else umma_commit<kCtas>(tmem_full_bar(acc));
                        }
                        ++ucount;
                    };
                    begin();
                    if (!ok) break;
                    const int last_steps = min(4, (p.K - (kb_first + kb_total - 1) * Cfg::BK + 63) / 64);
                    auto products = [&](int st, bool first, int steps) {
                        const uint64_t step = static_cast<uint64_t>(st * (Cfg::STAGE_BYTES >> 4));
                        const uint32_t sfa = tmem_base + Cfg::SCALE_AT + st * Cfg::SCALE_COLS, sfb = sfa + 8 + shift;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (k < steps) {
                                const uint32_t id = idesc0 | (k & 1 ? (2u << 4) | (2u << 29) : 0u);
                                umma_mxf4<kCtas>(lead, d_tmem, da0 + step + 2 * k, db0 + step + 2 * k, id, sfa + 4 * (k >> 1),
                                                 sfb + (k >> 1) * Cfg::B_TILES * 4, (first && k == 0) ? 0u : 1u);
                            }
                        }
                        if (lead) {
                            if constexpr (kPair) umma_commit_pair(empty_bar(st));
                            else umma_commit<kCtas>(empty_bar(st));
                        }
                    };
                    // Two k-blocks a turn: waiting, looking ahead and the loop take as long as half a k-block's products
                    // (8192^3, loops of a few ms: 204 us one by one, 187 us; 199-226 us in blocks of 0.15 s).
                    for (int kb = 0; kb < kb_total; kb += 2) {
                        const int s1 = s + 1 == STAGES ? 0 : s + 1, s2 = s1 + 1 == STAGES ? 0 : s1 + 1, s3 = s2 + 1 == STAGES ? 0 : s2 + 1;
                        const uint32_t ph1 = ph ^ (s1 == 0), ph2 = ph1 ^ (s2 == 0), ph3 = ph2 ^ (s3 == 0);
                        const bool two = kb + 1 < kb_total;
                        // an accumulator begins with a turn: what it sums is an even power of two of k-blocks
                        const bool next_acc = kLong && kb != 0 && (kb & (p.e.whole_kb - 1)) == 0;
                        if (next_acc) {
                            end();
                            begin();
                            if (!ok) break;
                        }
                        if (!ready)
                            ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, wc, kWaitFullStage) &&
                                                             (!two || mbar_wait(full_bar(s1), ph1, wc, kWaitFullStage)));
                        if (!ok) break;
                        tc_fence_after_sync();
                        if (two) {
                            // look at the next two now: the answer arrives while these two's products are issued
                            const bool next = mbar_test(full_bar(s2), ph2) && mbar_test(full_bar(s3), ph3);
                            products(s, kb == 0 || next_acc, 4);
                            products(s1, false, kb + 2 == kb_total ? last_steps : 4);
                            ready = __all_sync(0xffffffffu, next);
                            s = s2;
                            ph = ph2;
                        } else {
                            products(s, kb == 0 || next_acc, last_steps);
                            ready = false;
                            s = s1;
                            ph = ph1;
                        }
                    }
                    if (!ok) break;
                    end();
                }
            }
            __syncwarp();
        } else if (warp == 3) {
            // ------------------------------------------------------------------ TMA producer of the scales
            // A thread of its own: with the scales' copies in warp 0 its issue rate bounds the pipeline.
            if (lane == 0) {
                int s = 0;
                uint32_t ph = 0;
                bool ok = true;
                for (int unit = unit_first; ok && unit < num_units; unit += unit_stride) {
                    const Unit u = decode(unit);
                    // a CTA of a pair may own no rows of A: its scales are then those of the last rows
                    const int a_row = u.group * p.a_per_group * p.a_tile_rows + min(u.m0 / 128, p.a_tile_rows - 1);
                    const ScaleRows b_rows = scale_rows(first128[u.group], u.n0 - off[u.group], u.cols);
                    auto load_stages = [&](auto one_copy) {
                        const uint32_t bytes = one_copy ? Cfg::SF_BYTES : 1024 * (1 + b_rows.count);
                        for (int kb = 0; kb < u.kb; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0)) {
                            ok = mbar_wait(empty_bar(s), ph ^ 1u, wc, kWaitEmptyStage);
                            if (!ok) break;
                            const uint32_t at = smem_base + s * Cfg::STAGE_BYTES + Cfg::A_BYTES + Cfg::B_BYTES;
                            // two tiles along K (behind an odd last one: zeros) of every row of tiles that this tile's columns
                            // touch; what an earlier stage left in the place of another row belongs to no column of the products
                            mbar_arrive_expect_tx(scales_full_bar(s), bytes);
                            tma_load_3d(at, &tmSA, 0, 2 * (kb_first + kb), a_row, scales_full_bar(s));
                            tma_load_3d(at + 1024, &tmSB, 0, 2 * (kb_first + kb), b_rows.first, scales_full_bar(s));
                            if (Cfg::B_TILES == 2 && !one_copy && b_rows.count == 2)
                                tma_load_3d(at + 2048, &tmSB, 0, 2 * (kb_first + kb), b_rows.first + 1, scales_full_bar(s));
                        }
                    };
                    // Without groups the map of B's scales ends with the rows in use, and a copy takes all rows of a tile; with
                    // groups it spans the most rows that there can be, and a copy takes one (4100 x 1111 x 4128 that way: 25.3 ->
                    // 25.9 us).
                    if (!p.offsets) load_stages(std::true_type());
                    else load_stages(std::false_type());
                }
            }
            __syncwarp();
        }
    } else if (warp >= 12) {
        regs_dec<56>();
        // ------------------------------------------------------------------ scales: shared -> tensor memory
        const uint32_t quarter = static_cast<uint32_t>((warp & 3) * 32) << 16;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int unit = unit_first; ok && unit < num_units; unit += unit_stride) {
            const int turn = kBN < 128 ? scale_shift(decode(unit)) / 32 : 0;
            for (int kb = 0; kb < kb_total; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0)) {
                ok = mbar_wait(scales_full_bar(s), ph, wc, kWaitScales);
                ok = __all_sync(0xffffffffu, ok);  // tcgen05.st is warp-collective
                if (!ok) break;
                // the stage's columns of tensor memory are free: its loads were issued after the products that
                // last read them
                const uint8_t* tiles = smem_gen + s * Cfg::STAGE_BYTES + Cfg::A_BYTES + Cfg::B_BYTES + lane * 16;
                const uint32_t sfa = tmem_base + quarter + Cfg::SCALE_AT + s * Cfg::SCALE_COLS, sfb = sfa + 8;
                uint4 r[2 * (1 + Cfg::B_TILES)];
#pragma unroll
                for (int i = 0; i < 2 * (1 + Cfg::B_TILES); ++i) r[i] = *reinterpret_cast<const uint4*>(tiles + i * 512);
                if constexpr (kBN < 128) {  // one column of 32 rows is all that the tile uses
#pragma unroll
                    for (int i = 2; i < 4; ++i) r[i].x = turn == 0 ? r[i].x : turn == 1 ? r[i].y : turn == 2 ? r[i].z : r[i].w;
                }
                tmem_st_32x32b_x4(sfa, r[0]);
                tmem_st_32x32b_x4(sfa + 4, r[1]);
#pragma unroll
                for (int i = 0; i < Cfg::B_TILES; ++i) {
                    tmem_st_32x32b_x4(sfb + i * 4, r[2 + 2 * i]);
                    tmem_st_32x32b_x4(sfb + (Cfg::B_TILES + i) * 4, r[3 + 2 * i]);
                }
                tmem_wait_st();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (kPair) mbar_arrive_cluster_relaxed(full_bar(s), 0);
                    else mbar_arrive(full_bar(s));
                }
            }
        }
        __syncwarp();
    } else {
        regs_inc<200>();
        const int wg = (warp - 4) >> 2;
        run_epilogue<Epi, kBN, ACCS, kCtas, false, ACCS == 1 ? -1 : 0, kLong, false, kSplit ? 2 : 1>(
            p.e, wg, tmem_base, tmem_full_bar(0), tmem_empty_bar(0), wc, unit_first, unit_stride, num_units, split, decode);
    }

    // ---------------------------------------------------------------------- common exit
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    if constexpr (kPair || kSplit) cluster_sync_all();
    if (warp == 2) {
        tc_fence_after_sync();
        tmem_dealloc<kCtas>(tmem_base, Cfg::TMEM_COLS);
    }
}

}  // namespace b200
