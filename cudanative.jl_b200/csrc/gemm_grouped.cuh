// Grouped products with ragged sizes for sm_100a: the persistent TMA + tcgen05 pipeline of
// gemm_sm100.cuh over groups whose extent along one dimension is data on the device.
//
//   ragged N (kRaggedK = false)   D[:, s_e] = alpha * op(A_e) * B[:, s_e] + beta * C[:, s_e]
//   ragged K (kRaggedK = true)    D_e = alpha * A[:, s_e] * B[:, s_e]^T + beta * C_e
//
// with s_e = [offsets[e], offsets[e + 1]).  For a layer with one weight matrix per group the first is
// the forward product and the gradient of its inputs, the second the gradient of the weights.
//
// The sizes are never copied to the host.  Every CTA reads the offsets (at most kMaxGroups), checks
// them and, for ragged N, scans the number of tile columns of each group into shared memory; a work
// unit is then found by binary search.  A tile never crosses a group's border:
//   ragged N  columns of B behind the border are loaded (they exist, or read as zero behind the last
//             column of B) and multiplied, but not stored; the instruction's N is cut to the columns
//             that are left, rounded up to the instruction's granule, so that short groups cost what
//             they hold.  A NaN in a neighbour's column stays in that column.
//   ragged K  the last k-block of a group holds rows that belong to the next group.  Whole 16-row
//             steps behind the border are not issued; inside the last step the rows behind the border
//             are overwritten with zeros in shared memory, in A and in B (0 * NaN is NaN), by warp 3
//             between the arrival of the tile and its use.
//
// Roles and barriers are those of gemm_sm100.cuh (warp 0 producer, warp 1 MMA issuer, warp 2 tensor
// memory) with the epilogue of epilogue_sm100.cuh in warps 4-11; every wait is bounded.  Offsets that decrease or leave
// [0, total] are reported (report_bad_offsets) and the launch writes nothing.
#pragma once

#include "epilogue_sm100.cuh"
#include "ptx_sm100.cuh"

namespace b200 {

constexpr int kMaxGroups = 1024;

// Division of 0 .. 2^31 - 1 by a number that the host knows, as a product: every role places every tile of its CTA,
// three divisions one after the other (256 groups of 512 x 768, 1501 columns: 61 us with divisions, 57 so).
// q = (high(n * mul) + n) >> shift with mul = floor(2^32 (2^shift - d) / d) + 1 and shift = ceil(log2 d) (Granlund
// and Montgomery 1994); n + high(n * mul) stays below 2^32.
struct Divisor {
    uint32_t mul, shift;
    int d;
    __host__ static Divisor of(int d) {
        uint32_t shift = 0;
        while ((1ull << shift) < static_cast<unsigned long long>(d)) ++shift;
        const unsigned long long mul = (((1ull << shift) - d) << 32) / d + 1;
        return {static_cast<uint32_t>(mul), shift, d};
    }
};
__device__ __forceinline__ int operator/(int n, const Divisor& v) {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), v.mul) + static_cast<uint32_t>(n)) >> v.shift);
}

// Tile rows are walked down inside bands of `band` rows: CTAs that run together share panels in L2.
struct Raster {
    Divisor band, rows;  // rows of all the tiles of a matrix
    __host__ static Raster of(int band, int rows) { return {Divisor::of(band), Divisor::of(rows)}; }
};
// Row and column of tile `idx` of a matrix with `cols` columns of tiles.
__device__ __forceinline__ int2 place_tile(const Raster& r, int idx, int cols) {
    if (r.rows.d <= r.band.d) {
        const int col = idx / r.rows;
        return make_int2(idx - col * r.rows.d, col);
    }
    const int band = idx / (r.band.d * cols), row0 = band * r.band.d, in = idx - row0 * cols, rows = r.rows.d - row0;
    const int col = rows >= r.band.d ? in / r.band : in / rows;
    return make_int2(row0 + in - col * min(rows, r.band.d), col);
}

struct GroupedParams {
    int N, K;              // ragged N: N = columns of B, C, D; ragged K: K = columns of A and B
    int groups;
    int tiles_n;           // ragged K only (tile columns of one D_e)
    Divisor tiles;         // ragged K only: tiles of one D_e
    Raster raster;
    const int* offsets;
    int a_per_group;       // ragged N: 0 = one A for all groups
    int ab_bf16;
    EpilogueParams e;
    int* status;
    unsigned long long wait_budget_ns;
};

// How a result's sum over K is put together: from one accumulator; of a binary32 D from several (epilogue_sm100.cuh); of
// a 16-bit D from several where K is long.  The last is a kernel of its own, for the calls whose K or, for ragged K, whose
// longest possible group passes whole_kb(): in the first one it cost 5% on many short groups that never need it.
enum : int { kOneAccumulator = 0, kBinary32 = 1, kLongSums = 2 };

// k-blocks that one accumulator of a 16-bit D sums at most: 16384 products for binary16, 65536 for bfloat16, which leaves sums of
// one sign 1.1e-4 or 4.3e-4 off where the rounding that follows is up to 4.9e-4 or 3.9e-3.
__host__ __device__ constexpr int whole_kb(int d_fmt) { return d_fmt == 1 ? 256 : 1024; }

template <int kBN, bool kRaggedK, int kCtas, int kSums, int kSplit>
struct GroupedCfg {
    static constexpr int THREADS = 384;
    static constexpr int BM = 128;
    static constexpr int BK = 64;
    static constexpr int BN_LOCAL = kBN / kCtas;
    static constexpr int A_BYTES = BM * BK * 2;
    static constexpr int B_BYTES = BN_LOCAL * BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int BBOX = BN_LOCAL < 64 ? BN_LOCAL : 64;  // B rows per bulk load
    static constexpr int BBOX_BYTES = BBOX * BK * 2;
    static constexpr int GRANULE = kCtas == 2 ? 32 : 16;        // of the instruction's N
    static constexpr int PROMOTE_KB = 8;                        // k-blocks per accumulator of a binary32 D
    using Epi = EpilogueCfg<kBN>;
    static constexpr int TABLE_BYTES = (kRaggedK ? 1 : 2) * (kMaxGroups + 4) * 4;
    static constexpr int BAR_BYTES = 512;
    static constexpr int SCAN_AT = 384;  // among them, behind the barriers: scratch of the groups' scan, a sum per warp
    static constexpr int RECV_BYTES = kSplit == 2 ? 128 * kSplitRow * 4 : kSplit == 4 ? 128 * kBN * 4 : 0;
    static constexpr int BUDGET = 227 * 1024 - 1024 - BAR_BYTES - TABLE_BYTES - RECV_BYTES;
    static constexpr int STAGES = BUDGET / STAGE_BYTES > 8 ? 8 : BUDGET / STAGE_BYTES;
    static constexpr int TMEM_COLS = 2 * kBN < 32 ? 32 : 2 * kBN;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + RECV_BYTES + TABLE_BYTES + BAR_BYTES + 1024;
    static constexpr int NBARS = 4 * STAGES + 6;
    static_assert(kSplit != 2 || (kCtas == 1 && !kRaggedK && kBN == 32), "two share K: one-CTA tiles, one warp group");
    static_assert(kSplit != 4 || (kCtas == 1 && kBN == 64 && kSums == kBinary32), "four share K: one-CTA tiles, 16 columns each");
    static_assert(!kRaggedK || BN_LOCAL % 64 == 0, "MN-major B loads 64 columns per box");
    static_assert(STAGES >= 3 && SMEM_BYTES <= 227 * 1024, "shared memory");
    static_assert(8 * NBARS + 8 <= SCAN_AT && SCAN_AT + THREADS / 32 * 8 <= BAR_BYTES, "barriers, scratch");
};

// Offsets into shared memory, checked and, for kTiles, with an exclusive scan of the tile columns per
// group in `first` (groups + 1 entries); `first128`, where given, gets the same for tiles of 128.  No
// offsets: one group of all columns.  All kThreads threads; returns false when the offsets are no
// ascending sequence inside [0, total].
template <bool kTiles, int kThreads = 256>
__device__ __forceinline__ bool load_groups(const int* offsets, int groups, int total, int tile, int* off, int* first,
                                            unsigned long long* warp_sums, int* first128 = nullptr) {
    constexpr int PER = kMaxGroups / kThreads + 1;  // entries 0 .. groups
    const int t = threadIdx.x;
    if (!offsets) {
        if (t < 2) {
            off[t] = t ? total : 0;
            if (kTiles) first[t] = t ? (total + tile - 1) / tile : 0;
            if (first128) first128[t] = t ? (total + 127) / 128 : 0;
        }
        __syncthreads();
        return true;
    }
    bool bad = false;
    unsigned long long n[PER], sum = 0;  // tiles in the low half, tiles of 128 in the high one
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = t * PER + i;
        n[i] = 0;
        if (e <= groups) off[e] = offsets[e];
        if (e < groups) {
            const int a = offsets[e], b = offsets[e + 1];
            if (a < 0 || b < a || b > total) bad = true;
            else if (kTiles) n[i] = static_cast<unsigned long long>((b - a) / 128 + ((b - a) % 128 != 0)) << 32 | static_cast<unsigned>((b - a) / tile + ((b - a) % tile != 0));
        }
        sum += n[i];
    }
    if constexpr (kTiles) {
        unsigned long long incl = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, d);
            if ((t & 31) >= d) incl += v;
        }
        if ((t & 31) == 31) warp_sums[t >> 5] = incl;
        bad = __syncthreads_or(bad) != 0;
        unsigned long long base = incl - sum;
#pragma unroll
        for (int w = 0; w < kThreads / 32 - 1; ++w) base += w < (t >> 5) ? warp_sums[w] : 0ull;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = t * PER + i;
            if (e <= groups) {
                first[e] = static_cast<int>(base);
                if (first128) first128[e] = static_cast<int>(base >> 32);
            }
            base += n[i];
        }
        __syncthreads();
    } else {
        bad = __syncthreads_or(bad) != 0;
    }
    return !bad;
}

// The group that tile column q belongs to: the last e with first[e] <= q (empty groups share their
// successor's start and are stepped over).
__device__ __forceinline__ int find_group(const int* first, int groups, int q) {
    int lo = 0, hi = groups;  // first[lo] <= q < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= q) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int kBN, bool kAMn, bool kRaggedK, int kCtas, int kSums, int kSplit>
__global__ void __launch_bounds__(384, 1)
gemm_grouped_tcgen05(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const GroupedParams p) {
    using Cfg = GroupedCfg<kBN, kRaggedK, kCtas, kSums, kSplit>;
    constexpr bool kPromote = kSums == kBinary32;
    constexpr int STAGES = Cfg::STAGES;
    using Epi = typename Cfg::Epi;
    constexpr bool kPair = (kCtas == 2);
    constexpr bool kBMn = kRaggedK;  // ragged K: both operands have their columns along k
    static_assert(!kRaggedK || kAMn, "ragged K: A is M x K column-major");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    constexpr int kRecvAt = STAGES * Cfg::STAGE_BYTES;
    constexpr int kTableAt = kRecvAt + Cfg::RECV_BYTES;
    const uint32_t bar_base = smem_base + kTableAt + Cfg::TABLE_BYTES;
    int* off = reinterpret_cast<int*>(smem_gen + kTableAt);
    int* first = off + kMaxGroups + 4;
    uint8_t* bar_gen = smem_gen + kTableAt + Cfg::TABLE_BYTES;

    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto tail_full_bar = [&](int s) { return bar_base + 8u * (2 * STAGES + s); };   // a group's last k-block has landed here
    auto tail_ready_bar = [&](int s) { return bar_base + 8u * (3 * STAGES + s); };  // ... and its foreign rows are zero
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (4 * STAGES + a); };
    auto tmem_empty_bar = [&](int a) { return bar_base + 8u * (4 * STAGES + 2 + a); };
    auto split_bar = [&](int i) { return bar_base + 8u * (4 * STAGES + 4 + i); };  // partial sums: full, empty
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
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
            mbar_init(tail_full_bar(s), 1);
            mbar_init(tail_ready_bar(s), kCtas);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tmem_full_bar(a), 1);
            mbar_init(tmem_empty_bar(a), 8 * kCtas);
        }
        mbar_init(split_bar(0), 1);  // the receiver's arrive; it expects the sender's bytes
        mbar_init(split_bar(1), kSplit == 4 ? 16 : 4);  // four warps of the receiver, or of each of the four CTAs
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 2) tmem_alloc<kCtas>(smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::TMEM_COLS);
    tc_fence_before_sync();
    __syncthreads();
    if constexpr (kPair || kSplit > 1) cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    griddep_launch_dependents();
    griddep_wait();

    const bool offsets_ok = load_groups<!kRaggedK, Cfg::THREADS>(p.offsets, p.groups, kRaggedK ? p.K : p.N, kBN, off, first,
                                                   reinterpret_cast<unsigned long long*>(bar_gen + Cfg::SCAN_AT));
    if (!offsets_ok && threadIdx.x == 0) report_bad_offsets(p.status, p.groups);
    const int tiles_m = p.raster.rows.d;
    const int num_units = !offsets_ok ? 0 : kRaggedK ? p.groups * p.tiles.d : first[p.groups] * tiles_m;

    // Split the inner dimension when that shortens the longest CTA's work (counted in whole tiles).
    SplitParams split;
    if constexpr (kSplit == 4) {
        split.role = static_cast<int>(cluster_cta_rank());
        unit_first = blockIdx.x >> 2;
        unit_stride = gridDim.x >> 2;
    }
    if constexpr (kSplit == 2) {
        const int ctas = gridDim.x, kb_all = (p.K + Cfg::BK - 1) / Cfg::BK;
        const int whole = (num_units + ctas - 1) / ctas, halves = (num_units + ctas / 2 - 1) / (ctas / 2);
        if (kb_all >= 4 && halves < 2 * whole) {
            split.role = static_cast<int>(cluster_cta_rank());
            unit_first = blockIdx.x >> 1;
            unit_stride = ctas >> 1;
        }
    }
    if constexpr (kSplit > 1) {
        split.recv = reinterpret_cast<const float*>(smem_gen + kRecvAt);
        split.recv_addr = smem_base + kRecvAt;
        split.full_bar = split_bar(0);
        split.empty_bar = split_bar(1);
    }

    auto decode = [&](int unit) {
        Unit u;
        int idx, tn_count;
        if constexpr (kRaggedK) {
            u.group = unit / p.tiles;
            idx = unit - u.group * p.tiles.d;
            tn_count = p.tiles_n;
        } else {
            u.group = find_group(first, p.groups, unit / p.raster.rows);
            idx = unit - first[u.group] * tiles_m;
            tn_count = first[u.group + 1] - first[u.group];
        }
        const int2 tile = place_tile(p.raster, idx, tn_count);
        const int tn = tile.y;
        u.m0 = tile.x * (Cfg::BM * kCtas) + static_cast<int>(cta_rank) * Cfg::BM;
        const int o0 = off[u.group], o1 = off[u.group + 1];
        if constexpr (kRaggedK) {
            u.n0 = tn * kBN;
            u.cols = min(kBN, p.N - u.n0);
            u.k0 = o0;
            u.k_len = o1 - o0;
        } else {
            u.n0 = o0 + tn * kBN;
            u.cols = min(kBN, o1 - u.n0);
            u.k0 = 0;
            u.k_len = p.K;
        }
        u.kb0 = 0;
        u.kb = (u.k_len + Cfg::BK - 1) / Cfg::BK;
        if (kSplit > 1 && split.role >= 0) {  // this CTA's share, the last ones' may be short or empty
            const int share = (u.kb + kSplit - 1) / kSplit;
            u.kb0 = min(u.kb, split.role * share);
            u.kb = min(share, u.kb - u.kb0);
        }
        return u;
    };
    auto inst_n = [&](const Unit& u) { return (u.cols + Cfg::GRANULE - 1) / Cfg::GRANULE * Cfg::GRANULE; };
    // this CTA has the group's last k-block and its last 16-row step is ragged: it has to be padded with zeros
    auto needs_tail = [&](const Unit& u) { return kRaggedK && (u.k_len % 16) != 0 && u.kb > 0 && (u.kb0 + u.kb) * Cfg::BK >= u.k_len; };

    // registers: 3 x 168 a thread at launch = 56 + 2 x 224; a binary32 result's sums stay in them
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
                    const uint32_t bytes = Cfg::A_BYTES + boxes * Cfg::BBOX_BYTES;
                    const int kb1 = u.kb;
                    const int z = u.group * p.a_per_group;
                    // one tile column in this group: A is read once, B again and again
                    const bool a_once = !kRaggedK && first[u.group + 1] - first[u.group] == 1;
                    for (int kb = 0; kb < kb1; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0)) {
                        ok = mbar_wait(empty_bar(s), ph ^ 1u, wc, kWaitEmptyStage);
                        if (!ok) break;
                        const uint32_t sa = smem_base + s * Cfg::STAGE_BYTES;
                        const uint32_t sb = sa + Cfg::A_BYTES;
                        const int k0 = u.k0 + (u.kb0 + kb) * Cfg::BK;
                        if constexpr (kRaggedK) {
                            const bool tail = needs_tail(u) && kb + 1 == kb1;
                            if (tail) {
                                // lands on this CTA's own barrier; warp 3 passes it on to the MMA issuer
                                const uint32_t tb = tail_full_bar(s);
                                mbar_arrive_expect_tx(tb, bytes);
                                tma_load_2d(sa, &tmA, u.m0, k0, tb);
                                tma_load_2d(sa + 8192, &tmA, u.m0 + 64, k0, tb);
                                for (int i = 0; i < boxes; ++i) tma_load_2d(sb + i * Cfg::BBOX_BYTES, &tmB, nb0 + i * 64, k0, tb);
                                if (cta_rank == 0) mbar_arrive(full_bar(s));  // keeps the stage's phase in step
                            } else if constexpr (kPair) {
                                const uint32_t fb = mapa_shared(full_bar(s), 0);
                                if (cta_rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * bytes);
                                tma_load_2d_pair(sa, &tmA, u.m0, k0, fb);
                                tma_load_2d_pair(sa + 8192, &tmA, u.m0 + 64, k0, fb);
                                for (int i = 0; i < boxes; ++i) tma_load_2d_pair(sb + i * Cfg::BBOX_BYTES, &tmB, nb0 + i * 64, k0, fb);
                            } else {
                                const uint32_t fb = full_bar(s);
                                mbar_arrive_expect_tx(fb, bytes);
                                tma_load_2d(sa, &tmA, u.m0, k0, fb);
                                tma_load_2d(sa + 8192, &tmA, u.m0 + 64, k0, fb);
                                for (int i = 0; i < boxes; ++i) tma_load_2d(sb + i * Cfg::BBOX_BYTES, &tmB, nb0 + i * 64, k0, fb);
                            }
                        } else {
                            uint32_t fb = full_bar(s);
                            if constexpr (kPair) fb = mapa_shared(fb, 0);
                            if (cta_rank == 0) mbar_arrive_expect_tx(full_bar(s), kCtas * bytes);
                            auto load_a = [&](uint32_t dst, int x, int y) {
                                if constexpr (kPair) tma_load_3d_pair(dst, &tmA, x, y, z, fb);
                                else if (a_once) tma_load_3d_hint(dst, &tmA, x, y, z, fb, once);
                                else tma_load_3d(dst, &tmA, x, y, z, fb);
                            };
                            if constexpr (kAMn) {
                                load_a(sa, u.m0, k0);
                                load_a(sa + 8192, u.m0 + 64, k0);
                            } else {
                                load_a(sa, k0, u.m0);
                            }
                            for (int i = 0; i < boxes; ++i) {
                                if constexpr (kPair) tma_load_2d_pair(sb + i * Cfg::BBOX_BYTES, &tmB, k0, nb0 + i * Cfg::BBOX, fb);
                                else tma_load_2d(sb + i * Cfg::BBOX_BYTES, &tmB, k0, nb0 + i * Cfg::BBOX, fb);
                            }
                        }
                    }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------------------------ MMA issuer
            // The whole warp walks the loop and one lane issues: see umma_mxf4 in ptx_sm100.cuh.
            if (cta_rank == 0) {
                const uint32_t lead = elect_lane();
                const uint32_t idesc0 = make_idesc_f16_f32(Cfg::BM * kCtas, 0, kAMn ? 1 : 0, kBMn ? 1 : 0, p.ab_bf16 ? 1 : 0);
                const uint64_t da0 = kAMn ? make_smem_desc(smem_base, 8192, 1024, kSwizzle128B)
                                          : make_smem_desc(smem_base, 16, 1024, kSwizzle128B);
                const uint64_t db0 = kBMn ? make_smem_desc(smem_base + Cfg::A_BYTES, 8192, 1024, kSwizzle128B)
                                          : make_smem_desc(smem_base + Cfg::A_BYTES, 16, 1024, kSwizzle128B);
                constexpr uint32_t kStepA = (kAMn ? 2048 : 32) >> 4, kStepB = (kBMn ? 2048 : 32) >> 4;
                int s = 0;
                uint32_t ph = 0, tail_ph = 0, ucount = 0;
                bool ok = true, ready = false;
                for (int unit = unit_first; ok && unit < num_units; unit += unit_stride) {
                    const Unit u = decode(unit);
                    // an empty group has no accumulator
                    const int kb_total = __shfl_sync(0xffffffffu, u.kb, 0);
                    const uint32_t idesc = idesc0 | (static_cast<uint32_t>(__shfl_sync(0xffffffffu, inst_n(u), 0) >> 3) << 17);
                    // 16-row steps of the last k-block; whether it has to be padded with zeros first
                    const int last_steps = min(Cfg::BK / 16, (u.k_len - (u.kb0 + kb_total - 1) * Cfg::BK + 15) / 16);
                    const bool tail = needs_tail(u);
                    auto products = [&](int st, uint32_t acc, bool first, int steps) {
                        const uint32_t d_tmem = tmem_base + acc * kBN;
                        const uint64_t da = da0 + static_cast<uint64_t>(st * (Cfg::STAGE_BYTES >> 4));
                        const uint64_t db = db0 + static_cast<uint64_t>(st * (Cfg::STAGE_BYTES >> 4));
#pragma unroll
                        for (int k = 0; k < Cfg::BK / 16; ++k)
                            if (k < steps) umma_f16_warp<kCtas>(lead, d_tmem, da + k * kStepA, db + k * kStepB, idesc, (first && k == 0) ? 0u : 1u);
                        if (lead) {
                            if constexpr (kPair) umma_commit_pair(empty_bar(st));
                            else umma_commit<kCtas>(empty_bar(st));
                        }
                    };
                    auto wait_tail = [&](int st) {  // the last k-block's foreign rows are zero
                        // of a pair, one CTA's rows were cleared by ordinary stores in the other CTA and are read from here
                        bool here;
                        if constexpr (kPair) here = mbar_wait_cluster(tail_ready_bar(st), (tail_ph >> st) & 1u, wc, kWaitTail);
                        else here = mbar_wait(tail_ready_bar(st), (tail_ph >> st) & 1u, wc, kWaitTail);
                        const bool done = __all_sync(0xffffffffu, here);
                        tail_ph ^= 1u << st;
                        return done;
                    };
                    // Two k-blocks a turn: waiting, looking ahead and the loop take as long as half a k-block's products.
                    // An accumulator begins and ends with a turn: what it sums is an even power of two of k-blocks.
                    const int acc_mask = (kPromote ? Cfg::PROMOTE_KB : p.e.whole_kb) - 1;
                    for (int kb = 0; kb < kb_total; kb += 2) {
                        const uint32_t acc = ucount & 1u;
                        const int s1 = s + 1 == STAGES ? 0 : s + 1, s2 = s1 + 1 == STAGES ? 0 : s1 + 1, s3 = s2 + 1 == STAGES ? 0 : s2 + 1;
                        const uint32_t ph1 = ph ^ (s1 == 0), ph2 = ph1 ^ (s2 == 0), ph3 = ph2 ^ (s3 == 0);
                        const bool two = kb + 1 < kb_total, last = kb + 2 >= kb_total;
                        const bool begin = kb == 0 || (kSums != kOneAccumulator && (kb & acc_mask) == 0);
                        const bool end = last || (kSums != kOneAccumulator && ((kb + 2) & acc_mask) == 0);
                        if (begin) ok = __all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(acc), ((ucount >> 1) & 1u) ^ 1u, wc, kWaitTmemEmpty));
                        if (ok && !ready)
                            ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, wc, kWaitFullStage) &&
                                                             (!two || mbar_wait(full_bar(s1), ph1, wc, kWaitFullStage)));
                        if (ok && last && tail) ok = wait_tail(two ? s1 : s);
                        if (!ok) break;
                        tc_fence_after_sync();
                        if (two) {
                            // look at the next two now: the answer arrives while these two's products are issued
                            const bool next = mbar_test(full_bar(s2), ph2) && mbar_test(full_bar(s3), ph3);
                            products(s, acc, begin, Cfg::BK / 16);
                            products(s1, acc, false, last ? last_steps : Cfg::BK / 16);
                            ready = __all_sync(0xffffffffu, next);
                            s = s2;
                            ph = ph2;
                        } else {
                            products(s, acc, begin, last_steps);
                            ready = false;
                            s = s1;
                            ph = ph1;
                        }
                        if (lead && end) {
                            if constexpr (kPair) umma_commit_pair(tmem_full_bar(acc));
                            else umma_commit<kCtas>(tmem_full_bar(acc));
                        }
                        ucount += end ? 1u : 0u;
                    }
                }
            }
            __syncwarp();
        } else if (kRaggedK && warp == 3) {
            // ------------------------------------------------------------------ zeros behind a group's last row
            int s = 0;
            uint32_t tail_ph = 0;
            bool ok = true;
            for (int unit = unit_first; ok && unit < num_units; unit += unit_stride) {
                const Unit u = decode(unit);
                const int kb1 = u.kb;
                if (needs_tail(u)) {
                    const int st = (s + kb1 - 1) % STAGES;
                    ok = mbar_wait(tail_full_bar(st), (tail_ph >> st) & 1u, wc, kWaitTail);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tail_ph ^= 1u << st;
                    // a tile is boxes of 64 (m or n) x 64 k, each k one line of 128 bytes: the swizzle moves
                    // 16-byte pieces inside a line only, so whole lines can be cleared
                    const int rem = u.k_len - (u.kb0 + kb1 - 1) * Cfg::BK, end = (rem + 15) / 16 * 16;
                    const int boxes = 2 + (inst_n(u) / kCtas + 63) / 64;  // A's two come first, B's follow
                    uint8_t* tile = smem_gen + st * Cfg::STAGE_BYTES;
                    for (int box = 0; box < boxes; ++box)
                        for (int row = rem + lane / 8; row < end; row += 4)
                            *reinterpret_cast<uint4*>(tile + box * 8192 + row * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (kPair) mbar_arrive_cluster(tail_ready_bar(st), 0);
                        else mbar_arrive(tail_ready_bar(st));
                    }
                }
                s = (s + kb1) % STAGES;
            }
            __syncwarp();
        }
    } else {
        regs_inc<224>();
        const int wg = (warp - 4) >> 2;
        run_epilogue<Epi, kBN, 2, kCtas, kPromote && kSplit != 4, kPromote ? Cfg::PROMOTE_KB : 0, kSums == kLongSums, kRaggedK, kSplit>(
            p.e, wg, tmem_base, tmem_full_bar(0), tmem_empty_bar(0), wc, unit_first, unit_stride, num_units, split, decode);
    }

    // ---------------------------------------------------------------------- common exit
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    if constexpr (kPair || kSplit > 1) cluster_sync_all();
    if (warp == 2) {
        tc_fence_after_sync();
        tmem_dealloc<kCtas>(tmem_base, Cfg::TMEM_COLS);
    }
}

}  // namespace b200
