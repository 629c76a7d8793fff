// Forward of the sparse MLA attention over the paged cache of kv rows in 8 bits (smla_cache.cuh), for sm_100a.
//
// Everything that is said at smla_fwd_kernel about the pair of CTAs, the ring, the tensor memory and the work ranges holds here; this is
// what differs.
//   operands   kind::f8f6f4 UMMAs on the stored e4m3 numbers as they lie, for K and for V: nothing is converted on the way, and a
//              gathered row is 576 bytes instead of 1152.  The other side of either product is the sum of an e4m3 (hi) and an e5m2 number (lo), a UMMA
//              each, with instruction descriptors of their own: q = 2^e (hi + lo) with e from the row's largest magnitude.  A bf16 number has eight
//              significant bits; hi to the nearest leaves a whole number of at most eight of the last place, which the three bits of lo hold.
//              So hi + lo is q exactly for what is within 2^-13 of the row's largest, and within 2^-21 of the largest for the rest.
//              P = hi + lo with the heaviest P of a row between 2^11 and 2^12: within 2^-8 of P, as in bf16, down to 2^-17 of the heaviest, and
//              within 2^-25 of the heaviest below.  A row may have one heavy key and thousands of light ones that weigh something together, so the
//              light ones must not be cut off: with lo in e4m3, whose smallest number is 2^-9, and the heaviest P at 2^6, o lost up to a quarter of
//              itself.  Both forms take the same time.
//              An 8-bit UMMA takes 32 of K in the time of 16 in bf16, so two of them cost what one contraction in bf16 costs.
//   scales     of a key's page, s_j.  The logits are x_j = scale 2^e s_j (hi + lo) c_j.  V needs p_j s_j, and that is what is rounded:
//              P_j = 2^(x_j + log2 s_j - ref), so that the heaviest P_j are alike whatever the pages' scales are: with ref set the
//              heaviest is 2^11, and ref moves (and O is rescaled) when one comes above 2^12, the most that hi + lo holds.  The sum is over
//              p_j = P_j / s_j.  A scale is a power of two: only its exponent is used.
//   lse, o     o = sum P_j c_j / sum p_j, lse = ref + log2 sum p_j; so partial results combine as in bf16.
//   Q          is split by the softmax warps when the last logits of the query before are there.
//   producers  look up pages and scales as well, indices two tiles and pages one tile ahead of the gather; softmax reads (s, log2 s, 1 / s) of
//              its keys from shared memory.
// What lives in registers decides: a spill goes to the L2 here, the shared memory leaves the L1 nothing.  So waits are inlined and the split of
// Q is a call.  On the way here, 4096 queries x 128 heads x top-k 2048, us in short runs: terms in fp32 and indices, pages and scales looked up by every
// softmax warp, running maximum 2482; packed arithmetic, reference that lags, two producer warps 2250; four 1968 (the two left two of the
// four sub-partitions' ports idle); pages and scales by the producers 1962, 512 x 64 x 2048 315 -> 301.  Gathers by TMA (tile::gather4, four rows
// an instruction) 5270: about 65 cycles an instruction.  Now, in calls back to back, under the power cap: 2320 (1.0 PFLOP/s), in short runs 2030; 512 x 64
// 347 and 299; 3000 x 128 x 512 of short prompts 597 and 578.
// S [64 heads per CTA x 256 keys] takes five slots of [128 keys x 128 columns] (the fifth half full), O two slots for every 128 keys.
#pragma once
#include "smla_cache.cuh"

namespace smla {

struct CacheView {
    const uint8_t* values;        // [n_pages][page rows][576]
    const float* scales;          // [n_pages]
    const int* table;             // [n_req][max_pages]
    const __nv_bfloat16* q;       // [s_q, h_q, 576]
    int n_pages, page_shift, n_req, max_pages;
};
// The page that holds position `idx` of the query's request, -1 where there is none.  Everything that a table or an index could hold is
// turned away here: nothing outside the cache is read.
__device__ __forceinline__ int cached_page(const CacheView& c, int idx, int key, const QMeta& m, int causal) {
    const bool ok = key < m.topk_len && idx >= 0 && idx < m.kv_len && (!causal || idx <= m.q_pos) && m.kv_base >= 0 && m.kv_base < c.n_req &&
                    (idx >> c.page_shift) < c.max_pages;
    return ok ? __ldcg(c.table + static_cast<size_t>(m.kv_base) * c.max_pages + (idx >> c.page_shift)) : -1;
}

namespace fc {
constexpr int kSoftmaxWarps = 16;
constexpr int kProducerThreads = 128;
constexpr int kThreads = kSoftmaxWarps * 32 + kProducerThreads + 64;
constexpr int kIssueWarp = kThreads / 32 - 2, kForwardWarp = kThreads / 32 - 1;
constexpr int kParts = 8;                  // a head's 256 keys of a tile over eight warps
constexpr int kTileKeys = 256;             // per pair; 128 per CTA
constexpr int kSlotBytes = 16384;          // [128 keys x 128 columns]
constexpr int kStages = 6;
constexpr int kKSlots = 5;                 // 576 columns: four times 128 and 64
constexpr int kTerm = 64 * 128;            // hi or lo of [64 head rows x 128 columns]
constexpr int kOffQ = 0;                   // [4][hi, lo][kTerm], then 64 columns of hi and 64 of lo side by side
constexpr int kOffP = 9 * kTerm;           // [2 x 128 keys][hi, lo][kTerm]
constexpr int kOffRing = kOffP + 4 * kTerm;
constexpr int kOffRows = kOffRing + kStages * kSlotBytes;     // [3 tiles][256] cache rows, see the producers for their order
constexpr int kOffStat = kOffRows + 3 * kTileKeys * 4;        // [2 tile parities][8 key parts][64 heads] row maxima / sums
constexpr int kOffScale = kOffStat + 2 * kParts * 64 * 4;     // [3 tiles][s, log2 s, 1 / s][256 keys] of the scale of the key's page
constexpr int kOffQExp = kOffScale + 3 * 3 * kTileKeys * 4;   // [2 query parities][64 heads] 2^e of the row
constexpr int kOffMisc = kOffQExp + 2 * 64 * 4;
constexpr int kMiscBytes = 256;                               // barriers
constexpr int kSmemBytes = kOffMisc + kMiscBytes + 1024;      // + alignment slack
constexpr int kTmemO = 0, kTmemS = 256;
constexpr float kTop = 11.f, kLag = 1.f;   // log2 of the heaviest P where the reference has just been set, and how much heavier one may come
static_assert(kSmemBytes <= 232448, "shared memory of one SM");
constexpr int kMinQExp = -126;             // smallest 2^e of a row of Q, the smallest normal number (its inverse is one too)
// Steps of 32 keys up to the last slot in use of the iterator's tile; four of them share two slots of V.
__device__ __forceinline__ int v_steps(const TileIter<1>& it) { return (min(kTileKeys, it.n_cur - it.tile() * kTileKeys) + 31) >> 5; }
__device__ __forceinline__ int v_slots(int steps) { return 2 * ((steps + 3) >> 2); }
}  // namespace fc

// A row of Q (row r of the image at `image`) into hi and lo, by eight lanes, and its 2^e.  A row that holds a NaN or an infinity becomes NaN.
// (A call: what the softmax warps hold is put aside around it, once a query, and not spilled among the work of every tile.)
__device__ __noinline__ void split_row(const __nv_bfloat16* row, uint32_t image, uint32_t exps, int r) {
    using namespace fc;
    const int u = threadIdx.x & 7;
    const uint4* src = reinterpret_cast<const uint4*>(row) + u;
    uint4 v[9];
#pragma unroll
    for (int j = 0; j < 9; ++j) v[j] = __ldg(src + j * 8);
    uint32_t top = 0;                            // largest magnitude among even / odd columns, as bf16 bits
#pragma unroll
    for (int j = 0; j < 9; ++j)
        top = __vmaxu2(__vmaxu2(__vmaxu2(top, v[j].x & 0x7fff7fffu), __vmaxu2(v[j].y & 0x7fff7fffu, v[j].z & 0x7fff7fffu)), v[j].w & 0x7fff7fffu);
    top = max(top >> 16, top & 0xffffu) << 16;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool bad = top >= 0x7f800000u;
    const int e = bad ? 0 : scale_exp(top, kMinQExp);
    const float f = bad ? __int_as_float(0x7fffffff) : exp2_int(-e);
    if (u == 0) st_shared_f32(exps + r * 4, exp2_int(e));
    const uint64_t f2 = pack_f32x2(f, f);
    const uint32_t to = image + r * 128 + (u & 1) * 8;
#pragma unroll
    for (int j = 0; j < 9; ++j) {
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        uint64_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = mul_f32x2(pack_f32x2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u)), f2);
        uint32_t h[2], l[2];
        split_e4m3_e5m2x4<false>(x[0], x[1], &h[0], &l[0]);
        split_e4m3_e5m2x4<false>(x[2], x[3], &h[1], &l[1]);
        const int unit = (j & 1) * 4 + (u >> 1);
        const uint32_t to_hi = to + (j >> 1) * 2 * kTerm + ((unit ^ (r & 7)) << 4);
        const uint32_t to_lo = j < 8 ? to_hi + kTerm : to + 8 * kTerm + (((4 + unit) ^ (r & 7)) << 4);
        st_shared_v2(to_hi, h[0], h[1]);
        st_shared_v2(to_lo, l[0], l[1]);
    }
}

template <int HP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(fc::kThreads, 1)
smla_fwd_cached_kernel(const KParams p, const CacheView c) {
    using namespace fc;
    constexpr int NH = HP / 2;               // heads of this CTA (of the 64 rows the UMMAs compute)
    constexpr int kBusyWarps = NH / 4;       // with 64 heads a CTA's rows 32-63 do not exist: the warps of those lane quarters idle
    const uint32_t rank = cluster_ctarank();
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t s_base = smem_u32(smem);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffMisc);
    const uint32_t bar_full = smem_u32(bars);               // [kStages] slot landed (even CTA: in both CTAs)
    const uint32_t bar_empty = bar_full + 8 * kStages;      // [kStages] the UMMAs reading the slot finished
    const uint32_t bar_qfull = bar_empty + 8 * kStages;     // Q of the query split (even CTA: in both CTAs)
    const uint32_t bar_tfull = bar_qfull + 8;               // [2] S buffer complete
    const uint32_t bar_tempty = bar_tfull + 16;             // [2] (even CTA) both CTAs have read the S buffer
    const uint32_t bar_pfull = bar_tempty + 16;             // P of the tile written (even CTA: in both CTAs)
    const uint32_t bar_pv = bar_pfull + 8;                  // O += P V of the tile finished
    const uint32_t bar_scale = bar_pv + 8;                  // [3] scales of the tile written
    const uint32_t bar_drain = bar_scale + 24;                  // used only while winding down after an abort
    constexpr int kBars = 2 * kStages + 11;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffMisc + 8 * kBars);
    volatile int* s_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    WorkRange* range_s = reinterpret_cast<WorkRange*>(tmem_slot + 2);
    static_assert(8 * kBars + 8 + sizeof(WorkRange) <= kMiscBytes, "barrier area");
    const WaitCtx wc{p.g_err, s_abort, p.wait_limit, map_to_cta(smem_u32(tmem_slot + 1), rank ^ 1)};

    if (threadIdx.x == 0) {
        *s_abort = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(bar_full + 8 * i, kProducerThreads + (rank == 0 ? 1 : 0));   // + the odd CTA's forwarded arrival
            mbar_init(bar_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_tfull + 8 * i, 1);
            mbar_init(bar_tempty + 8 * i, 2 * kBusyWarps);
        }
        mbar_init(bar_qfull, kBusyWarps + (rank == 0 ? 1 : 0));      // + the odd CTA's forwarded arrival
        mbar_init(bar_pfull, kBusyWarps + (rank == 0 ? 1 : 0));      // likewise
        mbar_init(bar_pv, 1);
        for (int i = 0; i < 3; ++i) mbar_init(bar_scale + 8 * i, kProducerThreads);
        mbar_init(bar_drain, 1);
        fence_mbar_init();
    }
    const int n_rows = min(max(p.h_q - static_cast<int>(rank) * NH, 0), NH);      // of this CTA's heads; a multiple of 8
    for (int i = threadIdx.x; i < 9 * (64 - n_rows) * 8; i += kThreads) {        // the others: computed from zeros, never read
        const int j = i / ((64 - n_rows) * 8), r = i % ((64 - n_rows) * 8);
        *reinterpret_cast<uint4*>(smem + kOffQ + j * kTerm + n_rows * 128 + r * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
    if (warp == kIssueWarp) {
        tmem_alloc_2cta(smem_u32(tmem_slot), 512);
        tmem_relinquish_2cta();
    }
    if (!p.every_slot) pdl_wait();   // the prep kernel's slot counts
    const int total = find_range<kThreads>(p, blockIdx.x >> 1, gridDim.x >> 1, reinterpret_cast<int*>(smem + kOffStat), range_s);
    if (total >= 0 && rank == 0 && !p.every_slot) p.range_q[blockIdx.x >> 1] = make_int4(range_s->q, range_s->lo, total, 0);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();          // barriers of both CTAs are initialised before anyone signals across
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const WorkRange range = uniform_range(*range_s);
    const int n_tiles = range.end - range.begin;
    if (p.every_slot) pdl_wait();    // nothing of the caller's has been touched so far
    pdl_trigger();                   // (the tensor memory is this CTA's: see the dq kernel)

    if (warp >= kSoftmaxWarps && warp < kIssueWarp) {
        // ------------------------------------------------------------------ gather producers
        const int pt = threadIdx.x - kSoftmaxWarps * 32;
        constexpr int kRows = kProducerThreads / 8;          // rows that the producers copy side by side
        constexpr int kCopies = 128 / kRows;
        static_assert(kRows % 8 == 0, "a thread's rows share their swizzle");
        const uint64_t pol_keep = l2_policy_evict_last();
        // thread copies 16-byte unit uk of rows rk + 16 i of a slot's 128 keys
        const int uk = pt & 7, rk = pt >> 3;
        const uint32_t dst0 = s_base + kOffRing + rk * 128 + ((uk ^ (rk & 7)) << 4);
        const uint32_t rows = s_base + kOffRows;             // row of key k of 128 at [k % 16][k / 16]: a thread's eight in a line
        int s = 0;
        uint32_t ph = 1;                    // parity that means "slot free" for the current pass over the ring
        // keys pt and pt + 128 of every tile: the index two tiles ahead of the gather, its page one tile ahead
        constexpr int kKeys = kTileKeys / kProducerThreads;
        TileIter<1> it(p, range);
        QMeta qm = load_qmeta(p, range.q), qm_idx = qm;
        int idx[kKeys], page[kKeys], at_row[kKeys], tile_key = 0;
        int slots_idx = 0, slots_page = 0;   // slots of V that the tile of idx / of page has
        auto load_idx = [&]() {              // of the iterator's tile; on to the next one
            if (!it.more()) return;
            tile_key = it.tile() * kTileKeys + pt;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                const int key = tile_key + i * kProducerThreads;
                idx[i] = key < p.topk ? __ldg(p.indices + static_cast<size_t>(it.q) * p.topk + key) : -1;
            }
            slots_idx = v_slots(v_steps(it));
            qm_idx = qm;
            if (it.advance() && it.more()) qm = load_qmeta(p, it.q);
        };
        auto load_page = [&]() {             // of what load_idx has read
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                page[i] = cached_page(c, idx[i], tile_key + i * kProducerThreads, qm_idx, p.causal);
                at_row[i] = idx[i] & ((1 << c.page_shift) - 1);
            }
            slots_page = slots_idx;
        };
        load_idx();
        load_page();
        load_idx();
        const uint8_t* src[kCopies];
        uint32_t nb[kCopies];                // 0: the slot takes no part, read nothing and land zeros
        auto address = [&](uint32_t keys, int col) {
#pragma unroll
            for (int i = 0; i < kCopies; i += 4) {
                const int4 r = ld_shared_s32x4(keys + rk * (kCopies * 4) + i * 4);
                const int row[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    nb[i + k] = row[k] >= 0 ? 16u : 0u;
                    src[i + k] = c.values + static_cast<size_t>(max(row[k], 0)) * kDQK + (col + uk * 16);
                }
            }
        };
        auto fill = [&](int col, bool all) {
            mbar_wait_inline(bar_empty + 8 * s, ph, wc, kErrFwd + 31, kPollSleepNs);
            const uint32_t d = dst0 + s * kSlotBytes;
            if (all) {
#pragma unroll
                for (int i = 0; i < kCopies; ++i) cp_async16_zfill_hint(d + i * kRows * 128, src[i] + col, nb[i], pol_keep);
            }
            cp_async_mbar_arrive_noinc(bar_full + 8 * s);
            if (++s == kStages) {
                s = 0;
                ph ^= 1;
            }
        };
        int slots = 0, slots_next = 0;
        for (int n = -1; n < n_tiles; ++n, slots = slots_next) {              // K of tile n + 1, then V of tile n
            if (n + 1 < n_tiles) {
                // Three buffers: the one written now was last read two steps ago, before the previous step's barrier.  (Its scales were last
                // read for the P of tile n - 2, whose V has left the ring: it was followed there by more than the ring holds.)
                const int buffer = (n + 1) % 3;
                const uint32_t mine = rows + buffer * (kTileKeys * 4);
                float scale[kKeys];
                bool valid[kKeys];
#pragma unroll
                for (int i = 0; i < kKeys; ++i) {
                    const int key = pt + i * kProducerThreads;
                    valid[i] = page[i] >= 0 && page[i] < c.n_pages;
                    st_shared_s32(mine + (key >> 7) * 512 + key % kRows * (kCopies * 4) + key / kRows % kCopies * 4,
                                  valid[i] ? (page[i] << c.page_shift) + at_row[i] : -1);
                    scale[i] = valid[i] ? __ldcg(c.scales + page[i]) : 1.f;
                }
                slots_next = slots_page;
                load_page();
                load_idx();
                asm volatile("bar.sync 3, %0;" ::"n"(kProducerThreads) : "memory");
                address(mine + rank * 512, 0);
#pragma unroll
                for (int j = 0; j < kKSlots; ++j) fill(j * 128, j < kKSlots - 1 || uk < 4);
#pragma unroll
                for (int i = 0; i < kKeys; ++i) {
                    // The exponent alone, and not below 2^-100, so that p = P / s and sums of 2^15 of them do not overflow.  The log of a key that takes no part: -inf.
                    const int e = max((__float_as_int(scale[i]) >> 23 & 0xff) - 127, kMinScaleExp);
                    const uint32_t to = s_base + kOffScale + buffer * (3 * kTileKeys * 4) + (pt + i * kProducerThreads) * 4;
                    st_shared_f32(to, exp2_int(e));
                    st_shared_f32(to + kTileKeys * 4, valid[i] ? static_cast<float>(e) : __int_as_float(0xff800000));
                    st_shared_f32(to + 2 * kTileKeys * 4, exp2_int(-e));
                }
                mbar_arrive(bar_scale + 8 * buffer);
            }
            if (n >= 0) {
                const uint32_t mine = rows + n % 3 * (kTileKeys * 4);
#pragma unroll 1
                for (int g = 0; g < slots; g += 2) {
                    address(mine + g * 256, rank * 128);     // columns [256 block + 128 rank, + 128)
                    fill(0, true);
                    fill(256, true);
                }
            }
        }
    } else if (warp == kForwardWarp) {
        // ------------------------------------------------------------------ odd CTA: "my Q is split", "my P is written"
        // Plain stores of this CTA's softmax warps either way: released for the issuer at cluster scope, see smla_fwd_kernel.
        if (lane == 0 && rank == 1) {
            const uint32_t qfull_even = map_to_cta(bar_qfull, 0), pfull_even = map_to_cta(bar_pfull, 0);
            uint32_t qpar = 0;
            TileIter<1> it(p, range);
            bool new_query = true;
            for (int n = -1; n < n_tiles; ++n) {
                if (it.more()) {                              // tile n + 1
                    if (new_query) {
                        mbar_wait_inline(bar_qfull, qpar, wc, kErrFwd + 36);
                        fence_proxy_async_smem();
                        mbar_arrive_cluster_release(qfull_even);
                        qpar ^= 1;
                    }
                    new_query = it.advance();
                }
                if (n >= 0) {
                    mbar_wait_inline(bar_pfull, n & 1, wc, kErrFwd + 42);
                    tc_fence_after_sync();
                    fence_proxy_async_smem();
                    tc_fence_before_sync();
                    mbar_arrive_cluster_release(pfull_even);
                }
            }
        }
    } else if (warp == kIssueWarp) {
        if (elect_one()) {
            if (rank == 1) {
                // -------------------------------------------------------------- forward slot-full to the even CTA
                RingReader<kStages, false> ring(bar_full);
                const uint32_t full_even = map_to_cta(bar_full, 0);
                TileIter<1> it(p, range);
                int slots = 0, slots_next = 0;
                for (int n = -1; n < n_tiles; ++n, slots = slots_next) {
                    const bool k_tile = n + 1 < n_tiles;
                    const int todo = (k_tile ? kKSlots : 0) + slots;
                    for (int j = 0; j < todo; ++j) {
                        ring.wait(wc, kErrFwd + 37);
                        const uint32_t s = ring.slot;
                        ring.next();
                        fence_proxy_async_smem();    // (copies that the wait has seen complete: see smla_fwd_kernel)
                        mbar_arrive_cluster_relaxed(full_even + 8 * s);
                    }
                    if (k_tile) {
                        slots_next = v_slots(v_steps(it));
                        it.advance();
                    }
                }
            } else {
                // -------------------------------------------------------------- UMMA issuer for the pair
                constexpr uint32_t idesc_s = make_idesc_e4m3(128, 256, 0, 0);
                constexpr uint32_t idesc_o = make_idesc_e4m3(128, 256, 0, 1);      // V: d contiguous (MN-major)
                const uint64_t hi = make_smem_desc(0, 16, 1024, kSwizzle128) & 0xFFFFFFFF00000000ull;
                const uint32_t lo = static_cast<uint32_t>(make_smem_desc(0, 16, 1024, kSwizzle128));
                const uint32_t q_lo = lo + desc_addr(s_base + kOffQ), p_lo = lo + desc_addr(s_base + kOffP), r_lo = lo + desc_addr(s_base + kOffRing);
                RingReader<kStages, false> ring(bar_full);
                uint32_t qpar = 0;
                TileIter<1> it(p, range);
                bool new_query = true;
                uint32_t first_bits = 0;      // bit n & 1: tile n is its query's first in this range
                int steps = 0, steps_next = 0;
                for (int n = -1; n < n_tiles; ++n, steps = steps_next) {
                    if (n + 1 < n_tiles) {
                        // S of tile n + 1
                        const int t = n + 1, b = t & 1;
                        mbar_wait_inline(bar_tempty + 8 * b, ((t >> 1) & 1) ^ 1, wc, kErrFwd + 33);
                        if (new_query) {
                            mbar_wait_inline(bar_qfull, qpar, wc, kErrFwd + 32);
                            qpar ^= 1;
                        }
                        const uint32_t d = tmem + kTmemS + b * 128;
#pragma unroll 1
                        for (int j = 0; j < kKSlots; ++j) {
                            ring.wait(wc, kErrFwd + 34);
                            const uint32_t s = ring.slot;
                            ring.next();
                            fence_proxy_async_smem();        // the slot was written by cp.async, the tensor core reads it
                            tc_fence_after_sync();
                            const uint32_t a = q_lo + j * (2 * kTerm >> 4), bb = r_lo + s * (kSlotBytes >> 4);
                            // 32 bytes further along K = +2 in the address field; lo lies one kTerm (in the last slot 64 bytes) behind hi
                            const bool whole = j < kKSlots - 1;
                            const uint32_t to_lo = whole ? kTerm >> 4 : 64 >> 4;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                if (kk >= 2 && !whole) break;
                                umma_f8_ss_2cta(d, hi | (a + 2 * kk), hi | (bb + 2 * kk), idesc_s, (j | kk) != 0);
                                umma_f8_ss_2cta(d, hi | (a + to_lo + 2 * kk), hi | (bb + 2 * kk), idesc_s | kIdescAE5M2, 1);
                            }
                            umma_commit_2cta_mask(bar_empty + 8 * s, 3);
                        }
                        umma_commit_2cta_mask(bar_tfull + 8 * b, 3);
                        steps_next = v_steps(it);
                        first_bits = (first_bits & ~(1u << b)) | (static_cast<uint32_t>(new_query) << b);
                        new_query = it.advance();
                    }
                    if (n >= 0) {
                        // O += P V of tile n
                        const uint32_t acc0 = ((first_bits >> (n & 1)) & 1u) ^ 1u;
                        mbar_wait_inline(bar_pfull, n & 1, wc, kErrFwd + 39);
                        const int slots = v_slots(steps);
#pragma unroll 1
                        for (int g = 0; g < slots; ++g) {
                            ring.wait(wc, kErrFwd + 34);
                            const uint32_t s = ring.slot;
                            ring.next();
                            fence_proxy_async_smem();        // the slot was written by cp.async, the tensor core reads it
                            tc_fence_after_sync();
                            const uint32_t a = p_lo + (g >> 1) * (2 * kTerm >> 4), bb = r_lo + s * (kSlotBytes >> 4);
                            const uint32_t d = tmem + kTmemO + (g & 1) * 128;
                            const int todo = steps - 4 * (g >> 1);
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {   // 32 keys: 32 bytes along P's rows, 32 rows (4 KB) of V
                                if (kk >= todo) break;
                                umma_f8_ss_2cta(d, hi | (a + 2 * kk), hi | (bb + kk * (4096 >> 4)), idesc_o, (g >> 1 | kk) != 0 ? 1u : acc0);
                                umma_f8_ss_2cta(d, hi | (a + (kTerm >> 4) + 2 * kk), hi | (bb + kk * (4096 >> 4)), idesc_o | kIdescAE5M2, 1);
                            }
                            umma_commit_2cta_mask(bar_empty + 8 * s, 3);
                        }
                        umma_commit_2cta_mask(bar_pv, 3);
                    }
                }
                if (*s_abort) {   // winding down: nothing of this thread's may still be in the tensor pipe at dealloc
                    umma_commit_2cta_mask(bar_drain, 1);
                    mbar_wait_drain(bar_drain, 0, p.wait_limit);
                }
            }
        }
    } else if ((warp & 1) * 32 < NH) {
        // ------------------------------------------------------------------ softmax (one head, 32 keys of the tile per thread)
        const int quarter = warp & 3, cg = warp >> 2;
        const int part = (quarter >> 1) * 4 + cg;                // which 32 keys of the tile
        const int row = (quarter & 1) * 32 + lane;               // head row of this CTA
        const int head = static_cast<int>(rank) * NH + row;
        const bool real = head < p.h_q;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t tempty0 = map_to_cta(bar_tempty, 0);
        const uint32_t p_row = s_base + kOffP + (part >> 2) * 2 * kTerm + row * 128;
        const int bar_id = 1 + (quarter & 1);                    // the eight warps that share 32 rows
        const uint32_t stat = s_base + kOffStat + row * 4;       // + 256 for every part
        const uint32_t scale0 = s_base + kOffScale + part * 128;         // of this warp's keys; + 3 KB for every buffer
        const float ninf = __int_as_float(0xff800000);
        // Q into hi and lo: this warp's four of the 32 rows that its eight warps share, eight lanes a row.  (Rows r, r + 1, r + 4, r + 5: their
        // halves of the swizzled 128 bytes are different banks.)  The next query's replaces it when the last logits of this one are there.
        const int split_row_id = (quarter & 1) * 32 + (warp >> 2) * 8 + ((warp >> 1) & 1) * 2 + ((lane >> 3) & 1) + (lane >> 4) * 4;
        const bool splits = split_row_id < n_rows;                  // (alike in a warp)
        const int split_u = lane & 7;
        auto q_row = [&](int qg) { return c.q + (static_cast<size_t>(qg) * p.h_q + static_cast<int>(rank) * NH + split_row_id) * kDQK; };
        // `parity` of the query among the cluster's: another warp may still read the exponent of the query before
        auto split_q = [&](int qg, int parity) {
            if (splits) split_row(q_row(qg), s_base + kOffQ, s_base + kOffQExp + parity * 256, split_row_id);
            fence_proxy_async_smem();
            asm volatile("bar.sync %0, 256;" ::"r"(bar_id) : "memory");      // the exponents of the 32 rows
            if (lane == 0) mbar_arrive(bar_qfull);
        };
        TileIter<1> it(p, range);
        if (n_tiles > 0) {
            split_q(range.q, 0);
        }
        int q_parity = 1;                    // of the query that is split next
        bool new_query = true;
        float ref = ninf, sum = 0.f;         // reference of the row's exponentials (log2 units), sum over this thread's keys
        float q_scale = 0.f;                 // from the row's accumulated products to logits in log2 units, without the page's scale
        bool any_valid = false;              // the query has had a valid slot
        // A query's O leaves when the next tile's exponentials are done (see smla_fwd_kernel)
        bool pending = false, pend_whole = false;
        float pend_inv = 0.f;
        int pend_row = 0;                 // row of o, or slot of the partial results
        const uint32_t o_cols = tmem + lanes + kTmemO + cg * 32;         // this warp's 32 columns of either d-block
        auto write_out = [&]() {
            pending = false;
            // lanes 0-63: columns [256 block, + 128), lanes 64-127: [256 block + 128, + 128)
#pragma unroll 1
            for (int blk = 0; blk < 2; ++blk) {
                uint32_t o[32];
                tmem_ld_32x32(o_cols + blk * 128, o);
                tmem_ld_wait();
                const int col = blk * 256 + (quarter >> 1) * 128 + cg * 32;
                const size_t at = static_cast<size_t>(pend_row) * kDV + col;
                if (real && pend_whole) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            w[i] = pack_bf16x2(__uint_as_float(o[16 * e + 2 * i]) * pend_inv, __uint_as_float(o[16 * e + 2 * i + 1]) * pend_inv);
                        if ((reinterpret_cast<uintptr_t>(p.gout) & 31) == 0) {
                            st_global_v8(p.gout + at + 16 * e, w);
                        } else {
#pragma unroll
                            for (int v = 0; v < 2; ++v)
                                *reinterpret_cast<uint4*>(p.gout + at + 16 * e + 8 * v) = make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
                        }
                    }
                } else if (real) {
#pragma unroll
                    for (int v = 0; v < 4; ++v)      // [slot][8 columns][heads]: a warp's store is 1 KB in one piece
                        st_global_v8(p.part_o + ((static_cast<size_t>(pend_row) * (kDV / 8) + (col >> 3) + v) * HP + head) * 8, *reinterpret_cast<const uint32_t(*)[8]>(o + 8 * v));
                }
            }
        };
        int seg_begin = 0;
        for (int n = 0; n < n_tiles; ++n) {
            if (new_query) {
                ref = ninf;
                sum = 0.f;
                any_valid = false;
                seg_begin = it.pos;
                q_scale = ld_shared_f32(s_base + kOffQExp + ((q_parity ^ 1) * 64 + row) * 4) * p.scale_log2e;
                if (splits && it.q + 1 < p.q0 + p.nq) {          // (nine lines a row)
                    prefetch_l2(q_row(it.q + 1) + split_u * 64);
                    prefetch_l2(q_row(it.q + 1) + split_u * 64 + 64);
                }
            }
            const int qg = it.q, q_lo = it.lo, q_hi = it.hi;
            const bool last = it.last_of_query();
            const int seg_end = it.pos + 1;
            const bool next_query = it.advance();

            const int b = n & 1;
            const uint32_t scale_s = scale0 + n % 3 * (3 * kTileKeys * 4);
            mbar_wait_inline(bar_scale + 8 * (n % 3), n / 3 & 1, wc, kErrFwd + 43, kPollSleepNs);
            const uint32_t mask = __ballot_sync(0xffffffffu, ld_shared_f32(scale_s + kTileKeys * 4 + lane * 4) != ninf);
            const bool split = next_query && it.more();
            mbar_wait_inline(bar_tfull + 8 * b, (n >> 1) & 1, wc, kErrFwd + 38, kPollSleepNs);
            tc_fence_after_sync();
            if (split) {                 // these logits were the query's last reads of Q
                split_q(it.q, q_parity);
                q_parity ^= 1;
            }
            uint32_t sv[32];
            tmem_ld_32x32(tmem + lanes + kTmemS + b * 128 + cg * 32, sv);
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            // the S buffer has been read (tcgen05.wait::ld), which is all the issuer needs to know
            if (lane == 0) mbar_arrive_cluster_relaxed(tempty0 + 8 * b);
            // x + log2 s.  (The scales of q and of the page first: a large one of the page alone would take the products beyond fp32.)
            const uint64_t q2 = pack_f32x2(q_scale, q_scale);
            uint64_t y[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const ulonglong2 s4 = ld_shared_f32x4(scale_s + 16 * i), l4 = ld_shared_f32x4(scale_s + kTileKeys * 4 + 16 * i);
                y[2 * i] = fma_f32x2(pack_f32x2(__uint_as_float(sv[4 * i]), __uint_as_float(sv[4 * i + 1])), mul_f32x2(s4.x, q2), l4.x);
                y[2 * i + 1] = fma_f32x2(pack_f32x2(__uint_as_float(sv[4 * i + 2]), __uint_as_float(sv[4 * i + 3])), mul_f32x2(s4.y, q2), l4.y);
            }
            if (mask != 0xffffffffu) {                       // warp-uniform
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 v = unpack_f32x2(y[i]);
                    y[i] = pack_f32x2(mask >> (2 * i) & 1u ? v.x : ninf, mask >> (2 * i + 1) & 1u ? v.y : ninf);
                }
            }
            float m[2] = {ninf, ninf};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 v = unpack_f32x2(y[i]);
                m[i & 1] = max3_f32(m[i & 1], v.x, v.y);
            }
            st_shared_f32(stat + (b * kParts + part) * 256, fmaxf(m[0], m[1]));
            any_valid = bar_or(bar_id, 256, mask != 0u) || any_valid;
            float scale_o = 1.f;
            bool rescale = false;
            float top = ninf;
#pragma unroll
            for (int i = 0; i < kParts; ++i) top = fmaxf(top, ld_shared_f32(stat + (b * kParts + i) * 256));
            if (top - ref > kTop + kLag) {       // (first valid tile: ref is -inf, O and the sum are still empty)
                // Logits of 2^27 bits and more, in steps of 16 and more: no P above what hi + lo holds, wherever the difference is rounded to.
                const float lower = top - kTop, next = top - lower > kTop + kLag ? top : lower;
                rescale = ref > ninf;
                if (rescale) scale_o = ex2_approx(ref - next);
                ref = next;
            }
            const float neg = ref == ninf ? 0.f : -ref;
            sum *= scale_o;
            const uint64_t neg2 = pack_f32x2(neg, neg);
            uint64_t add = 0;
            uint32_t p_hi[8], p_lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const ulonglong2 inv = ld_shared_f32x4(scale_s + 2 * kTileKeys * 4 + 16 * i);
                uint64_t x[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 z = unpack_f32x2(add_f32x2(y[2 * i + k], neg2));
                    x[k] = pack_f32x2(ex2_approx(z.x), ex2_approx(z.y));
                    add = fma_f32x2(x[k], k ? inv.y : inv.x, add);
                }
                split_e4m3_e5m2x4<true>(x[0], x[1], &p_hi[i], &p_lo[i]);
            }
            {
                const float2 v = unpack_f32x2(add);
                sum += v.x + v.y;
            }
            // P of the previous tile has been consumed and O is at rest
            if (n > 0) mbar_wait_inline(bar_pv, (n - 1) & 1, wc, kErrFwd + 40, kPollSleepNs);
            tc_fence_after_sync();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t to = p_row + ((((part & 3) * 2 + u) ^ (row & 7)) << 4);
                st_shared_v4(to, p_hi[4 * u], p_hi[4 * u + 1], p_hi[4 * u + 2], p_hi[4 * u + 3]);
                st_shared_v4(to + kTerm, p_lo[4 * u], p_lo[4 * u + 1], p_lo[4 * u + 2], p_lo[4 * u + 3]);
            }
            fence_proxy_async_smem();
            if (pending) write_out();
            if (__any_sync(0xffffffffu, rescale)) {          // this warp's quarter of the columns of both d-blocks
#pragma unroll 1
                for (int blk = 0; blk < 2; ++blk) {
                    uint32_t o[32];
                    tmem_ld_32x32(o_cols + blk * 128, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * scale_o);
                    tmem_st_32x32(o_cols + blk * 128, o);
                }
                tmem_st_wait();
            }
            tc_fence_before_sync();
            __syncwarp();
            // Local arrival, forwarded by a thread of the odd CTA
            if (lane == 0) mbar_arrive(bar_pfull);

            if (last) {
                // ---- the query's (or the range's) last tile: lse now, o once its P V is done - or an unnormalised part of them
                const bool whole = seg_begin == q_lo && seg_end == q_hi;
                const uint32_t sums = stat + kParts * ((n + 1) & 1) * 256;
                st_shared_f32(sums + part * 256, sum);
                asm volatile("bar.sync %0, 256;" ::"r"(bar_id) : "memory");
                float total = 0.f;
#pragma unroll
                for (int i = 0; i < kParts; ++i) total += ld_shared_f32(sums + i * 256);
                asm volatile("bar.sync %0, 256;" ::"r"(bar_id) : "memory");      // the next tile's maxima go to the same place
                const int orow = qg * p.h_q + head;
                // partial results: slot 2 c for a range that starts inside the query, 2 c + 1 for one that starts at or before it
                const int slot = static_cast<int>(blockIdx.x >> 1) * 2 + (seg_begin == q_lo ? 1 : 0);
                if (real && part == 0) {
                    if (whole) p.lse_out[orow] = any_valid ? row_lse(ref, total) * p.lse_out_mult : no_slot_lse(p);
                    else p.part_ml[slot * HP + head] = make_float2(ref, any_valid ? total : kNoSlot);
                }
                pending = true;
                pend_whole = whole;
                pend_inv = any_valid ? 1.f / total : 0.f;        // no valid slot: O is 0
                pend_row = whole ? orow : slot;
            }
            new_query = next_query;
        }
        if (pending) {
            mbar_wait_inline(bar_pv, (n_tiles - 1) & 1, wc, kErrFwd + 41, kPollSleepNs);
            tc_fence_after_sync();
            write_out();
        }
    }
    abort_wind_down(s_abort);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();          // neither CTA leaves while the other may still signal it or read its operands
    if (warp == kIssueWarp) tmem_dealloc_2cta(tmem, 512);
}

}  // namespace smla
