// Device kernels around the paged cache of kv rows in 8 bits: the tables of a serving step (pages for new tokens, slot map, query
// table) and the write of new rows.  The attention that reads the cache is in smla_fwd_cached.cuh.
//
// The cache: values e4m3 [n_pages][page rows][576], scales fp32 [n_pages].  A page's rows share one scale, a power of two, so that going
// over to a larger scale moves exponents only (a number rounds again only where it becomes subnormal), and so that a stored number
// times its scale is a bf16 number exactly.  A slot is page * page rows + row.
//
// These kernels and the forward may come up under one another's tails.  What one of them changes in place (tables, free pages, scales, values)
// is read past the L1: a line of it that a block of the kernel before has brought there need not hold what another block of that kernel wrote.
#pragma once
#include <cuda_fp16.h>

#include "smla_kernels.cuh"

namespace smla {

constexpr int kMinScaleExp = -100;          // rows are stored with a scale of 2^-100 at least
constexpr int kMaxPageRows = 128;

// The smallest e >= min_exp with amax <= 448 * 2^e (448: the largest e4m3 number, 1.75 * 2^8), for a finite amax >= 0.
__device__ __forceinline__ int scale_exp(uint32_t amax_bits, int min_exp) {
    const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, min_exp);
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

// Four numbers -> e4m3, nearest even, the first in the low byte.  What is beyond 448 becomes 448, a NaN stays one.
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
// Packed halves: two numbers -> e4m3, nearest even, and back.
__device__ __forceinline__ uint32_t cvt_e4m3x2_f16x2(__half2 v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&v)));
    return r;
}
__device__ __forceinline__ __half2 cvt_f16x2_e4m3x2(uint32_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(v)));
    return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ uint32_t half2_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// Two numbers as the sum of an e4m3 number (hi) and an e5m2 number (lo) each: hi is x to four significant bits and lo three bits of what that
// leaves, at most half of hi's last place.  For |x| <= 448: to eight bits from 2^-6 on, exactly where x has no more than eight, and to within 2^-14
// below.  With kLarge for 0 <= x <= 2^12: from 2^8 on, where hi would not reach, c is x to three bits, hi takes four of what c leaves, and x - hi to
// three bits is c again.  An e5m2 number is the upper byte of a half; *lo: halves, whose upper bytes are lo.  (Eleven bits of a half, and its
// smallest numbers of 2^-24, are more than what is kept.)
template <bool kLarge> __device__ __forceinline__ uint32_t split_e4m3_e5m2(uint64_t x01, uint32_t* lo) {
    const float2 a = unpack_f32x2(x01);
    const __half2 x = __floats2half2_rn(a.x, a.y);
    __half2 main = x;
    if constexpr (kLarge) {
        const uint32_t c = (half2_bits(x) + 0x00800080u) & 0xff00ff00u & __hge2_mask(x, __floats2half2_rn(256.f, 256.f));
        main = __hsub2(x, *reinterpret_cast<const __half2*>(&c));
    }
    const uint32_t hi = cvt_e4m3x2_f16x2(main);
    *lo = half2_bits(__hsub2(x, cvt_f16x2_e4m3x2(hi))) + 0x00800080u;
    return hi;
}
template <bool kLarge> __device__ __forceinline__ void split_e4m3_e5m2x4(uint64_t x01, uint64_t x23, uint32_t* hi, uint32_t* lo) {
    uint32_t l01, l23;
    const uint32_t h01 = split_e4m3_e5m2<kLarge>(x01, &l01), h23 = split_e4m3_e5m2<kLarge>(x23, &l23);
    *hi = h01 | h23 << 16;
    *lo = __byte_perm(l01, l23, 0x7531);
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t v) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(v)));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// =============================================================================================
// Tables of a step.
//
// Every block adds up the requests' pages and tokens itself (8 bytes a request out of L2) and then takes its share of the tokens and
// of the pages that change hands, so one launch does it, with no prefix sums in memory.  That needs no order between the blocks: what is
// read (free_pages below free_count, the block table's entries of pages that requests had before the call) is not written by any
// of them.  A page that is given back and taken again in the same call is looked up in the row of the request that gives it.
// A request whose last tokens are dropped keeps its pages and writes its new tokens over them; what it does not need any more it gives back, and then it
// takes none.
// Bound by latency: a launch, two dependent loads and three block sums.
// =============================================================================================
struct CachePlanArgs {
    const int *kv_len, *new_len, *free_count;
    const int* rejected;          // (kRejects)
    int *table, *free_pages;
    int *slots, *kv_len_out, *free_count_out, *admitted;
    int4* meta;
    int n_req, max_pages, n_free, page_shift, max_tokens, topk;
};
constexpr int kCachePlanThreads = 512;
constexpr int kMaxCacheRequests = 8192;

// The largest i < n with a[i] <= x, for a[0] = 0 <= x and a[] not decreasing.
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Sum of one value per thread over the lower-numbered threads, not above `cap`, for values of 0 .. cap and a cap below 2^30; *total: over all.
__device__ __forceinline__ int block_exclusive_capped_sum(int v, int cap, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl = min(incl + up, cap);
    }
    const int left = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < n_warps; ++w) {
        if (w == warp) before = all;
        all = min(all + warp_sums[w], cap);
    }
    __syncthreads();
    *total = all;
    return lane ? min(before + left, cap) : before;
}

template <bool kRejects> __global__ void __launch_bounds__(kCachePlanThreads) smla_cache_plan_kernel(const CachePlanArgs a) {
    extern __shared__ int plan_smem[];
    __shared__ int warp_sums[kCachePlanThreads / 32];
    int* first = plan_smem;                       // [n_req + 1] tokens of the requests before, at most max_tokens + 1
    int* len = first + a.n_req + 1;               // [n_req] tokens that stay, ~ of them for a request that gets no row
    int* needx = len + a.n_req;                   // [n_req + 1] new pages asked for by the requests before
    int* backx = needx + a.n_req + 1;             // [n_req + 1] pages given back by the requests before
    pdl_wait();
    pdl_trigger();
    const int page = 1 << a.page_shift, cap = a.max_tokens + 1;
    const int n_free = min(max(__ldg(a.free_count), 0), a.n_free);
    const int per = (a.n_req + kCachePlanThreads - 1) / kCachePlanThreads;
    const int i0 = min(static_cast<int>(threadIdx.x) * per, a.n_req), i1 = min(i0 + per, a.n_req);
    const int room = a.max_pages << a.page_shift;                      // (below 2^31: checked on the host)
    auto length = [&](int i) { return min(max(__ldg(a.kv_len + i), 0), room); };
    auto pages_of = [&](int tokens) { return (tokens + page - 1) >> a.page_shift; };
    auto stays = [&](int i, int old) { return kRejects ? old - min(max(__ldg(a.rejected + i), 0), max(old, 0)) : old; };
    int tokens = 0;
    for (int i = i0; i < i1; ++i) tokens = min(tokens + min(max(__ldg(a.new_len + i), 0), cap), cap);
    int n_back, n_tokens, n_need, n_taken;
    const int first0 = block_exclusive_capped_sum(tokens, cap, warp_sums, &n_tokens);
    // what request i asks for beyond the pages it has, given the tokens before it; -1: it cannot have its rows whatever is free.  *give: pages that
    // it gives back
    auto need_of = [&](int i, int n, int before, int* give) {
        const int old = __ldg(a.kv_len + i), keep = stays(i, old);
        *give = n < 0 ? pages_of(length(i)) : 0;
        if (n < 0 || old < 0 || old > room || n > room - keep || before + min(n, cap) > a.max_tokens) return -1;
        const int more = pages_of(keep + n) - pages_of(old);
        *give = max(-more, 0);
        return max(more, 0);
    };
    int need = 0, back = 0;
    for (int i = i0, f = first0; i < i1; ++i) {
        const int n = __ldg(a.new_len + i);
        int give;
        need += max(need_of(i, n, f, &give), 0);
        back += give;
        f = min(f + min(max(n, 0), cap), cap);
    }
    const int need0 = block_exclusive_sum(need, warp_sums, &n_need);
    const int back0 = block_exclusive_sum(back, warp_sums, &n_back);
    const int stack = n_free + n_back;
    int taken = 0;
    for (int i = i0, f = first0, u = need0, b = back0; i < i1; ++i) {
        int give;
        const int n = __ldg(a.new_len + i), old = stays(i, length(i)), want = need_of(i, n, f, &give);
        const bool granted = want >= 0 && (want == 0 || u + want <= stack);
        first[i] = f;
        len[i] = granted ? old : ~old;
        needx[i] = u;
        backx[i] = b;
        if (blockIdx.x == 0) {
            a.kv_len_out[i] = n < 0 ? 0 : granted ? old + n : __ldg(a.kv_len + i);
            a.admitted[i] = granted ? n : 0;
        }
        f = min(f + min(max(n, 0), cap), cap);
        u += max(want, 0);
        if (granted) taken += want;
        b += give;
    }
    if (threadIdx.x == 0) first[a.n_req] = n_tokens;
    block_exclusive_sum(taken, warp_sums, &n_taken);           // (its barriers: the tables are whole)
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.free_count_out = min(stack - n_taken, a.n_free);
    // page v of the ones given back: all of a request that ends, the ones behind its last token of a request that goes on
    auto given_back = [&](int v) {
        const int i = last_not_above(backx, a.n_req, v), from = !kRejects || len[i] < 0 ? 0 : pages_of(len[i] + (first[i + 1] - first[i]));
        return __ldcg(a.table + static_cast<size_t>(i) * a.max_pages + (from + v - backx[i]));
    };
    // place s of the stack of free pages, the pages given back on top
    auto stacked = [&](int s) { return s < n_free ? __ldcg(a.free_pages + s) : given_back(s - n_free); };
    auto pages_held = [&](int i) { return pages_of(kRejects ? length(i) : len[i]); };      // by a request that gets its rows
    const int at = blockIdx.x * kCachePlanThreads + threadIdx.x, step = gridDim.x * kCachePlanThreads;
    for (int t = at; t < a.max_tokens; t += step) {
        int slot = -1;
        int4 m = make_int4(0, 0, 0, 0);
        if (t < n_tokens) {
            const int i = last_not_above(first, a.n_req, t), old = len[i];
            if (old >= 0) {
                const int pos = old + t - first[i], k = pos >> a.page_shift, have = pages_held(i);
                const int pg = k < have ? __ldcg(a.table + static_cast<size_t>(i) * a.max_pages + k) : stacked(stack - 1 - (needx[i] + k - have));
                slot = pg * page + (pos & (page - 1));
                m = make_int4(i, old + (first[i + 1] - first[i]), pos, a.topk);
            }
        }
        a.slots[t] = slot;
        a.meta[t] = m;
    }
    for (int u = at; u < n_taken; u += step) {
        const int i = last_not_above(needx, a.n_req, u);
        a.table[static_cast<size_t>(i) * a.max_pages + pages_held(i) + (u - needx[i])] = stacked(stack - 1 - u);
    }
    for (int v = at; v < n_back && n_free + v < a.n_free; v += step) a.free_pages[n_free + v] = given_back(v);
}

// =============================================================================================
// New rows into the cache.
//
// One block per page that the call names: it finds all rows of the call that go to the page, their largest finite magnitude, the page's
// scale, and writes.  Rows kept by a page whose scale grows are brought over to the new scale in the same block.
// The first row of a run (neighbours in the call that name one page) speaks for the run; a page may come up in several runs, whose
// first one does the work for all.  Up to kAppendDirect rows every row has a block, which looks through the whole slot map; beyond that
// a first kernel lists the runs, and the blocks go through the list.
// Bound by HBM (1152 bytes read and 576 written a row) for prompts, by latency for the rows of a decoding step.  65536 rows in 37 requests, pages
// of 128: 61 us with a block a page, 42 with two blocks of a cluster that exchange their maxima (2.7 TB/s; the same rows again and again, 36 us).
// On those: 46 with four blocks, whose lists and tables to look through are the larger part of their instructions, 58 - 65 with the rows held in
// registers in between, fewer blocks at a time.  Pages of 64 / 32 / 16: 32 / 42 / 96 us, a run's lookups for fewer rows.
struct CacheAppendArgs {
    const __nv_bfloat16* kv;
    long long kv_stride;          // elements from row to row
    uint8_t* values;
    float* scales;
    const int* slots;
    int n_rows, n_pages, page_shift;
    int2* runs;                   // [lists][list_len] {page, first row}
    int* counts;                  // [lists]
    int n_lists, list_len;
};
constexpr int kAppendUnits = kDQK / 8;        // 16 bytes of a bf16 row, 8 bytes of a stored one
constexpr int kAppendSide = 4;                // rows that a block works on side by side
constexpr int kAppendThreads = kAppendSide * kAppendUnits;
static_assert(kAppendThreads % 32 == 0 && kAppendThreads >= kMaxPageRows, "whole warps, a thread for a page's row");
// Below, whatever the rows are: a list helps runs of many rows and is costly for single ones, and the host does not know which they are.  Pages of
// 64, direct / listed, us: 2048 rows of as many requests 8.1 / 57, 4096 17.5 / 148, 8192 46 / 415; of prompts of 512 rows 9.0 / 9.6, 11.3 / 9.8,
// 17.0 / 11.4, 16384 25.9 / 12.2.
constexpr int kAppendDirect = 8192;
constexpr int kAppendListLen = 1024;
constexpr int kAppendMaxLists = 512;
constexpr int kAppendBlockRows = 64;         // rows of a page that a block of the listed form takes

__device__ __forceinline__ int append_page_of(const CacheAppendArgs& a, int slot) {
    const int page = slot >> a.page_shift;
    return slot >= 0 && page < a.n_pages ? page : -1;
}
__device__ __forceinline__ bool append_run_begins(const CacheAppendArgs& a, int t, int page) {
    return page >= 0 && (t == 0 || append_page_of(a, __ldg(a.slots + t - 1)) != page);
}

__global__ void __launch_bounds__(1024) smla_cache_runs_kernel(const CacheAppendArgs a) {
    __shared__ int n;
    if (threadIdx.x == 0) n = 0;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    const int t0 = blockIdx.x * a.list_len, t1 = min(t0 + a.list_len, a.n_rows);
    for (int t = t0 + threadIdx.x; t < t1; t += 1024) {
        const int page = append_page_of(a, __ldg(a.slots + t));
        if (append_run_begins(a, t, page)) a.runs[t0 + atomicAdd(&n, 1)] = make_int2(page, t);     // (in any order)
    }
    __syncthreads();
    if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

struct AppendShared {
    int win[kMaxPageRows];        // row of the call that goes to row r of the page, -1: none
    int rows[kMaxPageRows];       // the page's rows that get one
    int n_rows, earlier, end;
    uint32_t warp_max[kAppendThreads / 32];
};

// The largest magnitude of even and odd columns so far and of eight more, as two sets of bf16 bits.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t top, const uint4& v) {
    return __vmaxu2(__vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu)), v.w & 0x7fff7fffu);
}
// The same for a page that has seen something not finite: over what is.
__device__ __forceinline__ uint32_t finite_max_bf16x2(uint32_t top, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t lo = w[k] & 0x7fffu, hi = w[k] & 0x7fff0000u;
        top = __vmaxu2(top, (lo < 0x7f80u ? lo : 0u) | (hi < 0x7f800000u ? hi : 0u));
    }
    return top;
}
// Eight columns as they are stored.  An infinity is stored as a NaN: the format has none, and it has no place among finite numbers.
__device__ __forceinline__ uint2 append_cvt(const uint4& v, float inv, bool all_finite) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const uint64_t inv2 = pack_f32x2(inv, inv);
    float2 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u)), inv2));
    if (!all_finite) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if ((w[k] & 0x7fffu) >= 0x7f80u) x[k].x = __uint_as_float(0x7fffffffu);
            if ((w[k] & 0x7fff0000u) >= 0x7f800000u) x[k].y = __uint_as_float(0x7fffffffu);
        }
    }
    return make_uint2(cvt_e4m3x4(x[0].x, x[0].y, x[1].x, x[1].y), cvt_e4m3x4(x[2].x, x[2].y, x[3].x, x[3].y));
}
// Rows [r0, r1) that the page keeps go over to its new scale.
__device__ __forceinline__ void append_rescale(const AppendShared& sh, uint8_t* base, int r0, int r1, float ratio) {
    for (int u = r0 * (kDQK / 16) + threadIdx.x; u < r1 * (kDQK / 16); u += kAppendThreads) {
        if (sh.win[u / (kDQK / 16)] >= 0) continue;
        uint4* at = reinterpret_cast<uint4*>(base + static_cast<size_t>(u) * 16);
        const uint4 v = __ldcg(at);
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 lo = e4m3x2_to_float2(w[k] & 0xffffu), hi = e4m3x2_to_float2(w[k] >> 16);
            w[k] = cvt_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Largest magnitude that the block's threads have seen, as bf16 bits; in every thread, behind a barrier.
__device__ __forceinline__ uint32_t append_block_max(uint32_t top, AppendShared& sh) {
    top = __reduce_max_sync(0xffffffffu, max(top >> 16, top & 0xffffu));
    if ((threadIdx.x & 31) == 0) sh.warp_max[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, sh.warp_max[w]);
    return top;
}

// The page's rows are known (win); quantise and write them.
__device__ __forceinline__ void append_write_page(const CacheAppendArgs& a, int page, AppendShared& sh) {
    const int page_rows = 1 << a.page_shift;
    if (static_cast<int>(threadIdx.x) < page_rows && sh.win[threadIdx.x] >= 0) sh.rows[atomicAdd(&sh.n_rows, 1)] = threadIdx.x;
    const float old = __ldcg(a.scales + page);
    __syncthreads();
    const int slot = threadIdx.x / kAppendUnits, unit = threadIdx.x % kAppendUnits, n = sh.n_rows;
    auto source = [&](int i) { return __ldg(reinterpret_cast<const uint4*>(a.kv + static_cast<long long>(sh.win[sh.rows[i]]) * a.kv_stride) + unit); };
    uint32_t top = 0;
#pragma unroll 4
    for (int i = slot; i < n; i += kAppendSide) top = max_bf16x2(top, source(i));
    top = append_block_max(top, sh);
    const bool all_finite = top < 0x7f80u;
    if (!all_finite) {
        top = 0;
        __syncthreads();
        for (int i = slot; i < n; i += kAppendSide) top = finite_max_bf16x2(top, source(i));
        top = append_block_max(top, sh);
    }
    const float wanted = exp2_int(scale_exp(top << 16, kMinScaleExp));
    const bool anew = sh.win[0] >= 0;             // its first row is written: what it held belongs to nobody
    const float scale = anew ? wanted : fmaxf(old, wanted);
    uint8_t* base = a.values + static_cast<size_t>(page) * page_rows * kDQK;
    if (!anew && scale > old) append_rescale(sh, base, 0, page_rows, old / scale);
    if (threadIdx.x == 0) a.scales[page] = scale;
    const float inv = 1.f / scale;
#pragma unroll 4
    for (int i = slot; i < n; i += kAppendSide)
        *reinterpret_cast<uint2*>(base + static_cast<size_t>(sh.rows[i]) * kDQK + unit * 8) = append_cvt(source(i), inv, all_finite);
}

__device__ __forceinline__ void append_clear(AppendShared& sh) {
    if (threadIdx.x < kMaxPageRows) sh.win[threadIdx.x] = -1;
    if (threadIdx.x == 0) sh.n_rows = sh.earlier = 0;
    __syncthreads();
}

__global__ void __launch_bounds__(kAppendThreads) smla_cache_append_kernel(const CacheAppendArgs a) {
    __shared__ AppendShared sh;
    const int row_mask = (1 << a.page_shift) - 1;
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x, page = append_page_of(a, __ldg(a.slots + t));
    if (!append_run_begins(a, t, page)) return;
    append_clear(sh);
#pragma unroll 4
    for (int i = threadIdx.x; i < a.n_rows; i += kAppendThreads) {
        const int slot = __ldg(a.slots + i);
        if (append_page_of(a, slot) == page) {
            if (i < t) sh.earlier = 1;
            atomicMax(&sh.win[slot & row_mask], i);
        }
    }
    __syncthreads();
    if (sh.earlier) return;                       // the page's first run does it
    append_write_page(a, page, sh);
}

// The blocks of a cluster share a page, 64 rows each.  They read them twice, the second time out of the L2: what holds them in between (32
// registers a thread) halves the blocks that are in place on an SM, and a page's way is a chain of a dozen latencies.
__global__ void __launch_bounds__(kAppendThreads, 6) smla_cache_append_listed_kernel(const CacheAppendArgs a) {
    __shared__ AppendShared sh;
    __shared__ int before[kAppendMaxLists + 1];   // runs in the lists before
    __shared__ __align__(16) uint32_t page_max[2][4];            // [parity of the page]
    const int row_mask = (1 << a.page_shift) - 1, page_rows = row_mask + 1;
    const int n_blocks = cluster_nctas(), rank = cluster_ctarank();
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x < 32) {
        int carry = 0;
        for (int l0 = 0; l0 < a.n_lists; l0 += 32) {
            const int l = l0 + threadIdx.x, c = l < a.n_lists ? __ldcg(a.counts + l) : 0;
            int incl = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, o);
                if (static_cast<int>(threadIdx.x) >= o) incl += up;
            }
            if (l < a.n_lists) before[l] = carry + incl - c;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (threadIdx.x == 0) before[a.n_lists] = carry;
    }
    __syncthreads();
    const int n_runs = before[a.n_lists];
    auto run = [&](int g) {
        const int l = last_not_above(before, a.n_lists, g);
        return __ldcg(a.runs + static_cast<size_t>(l) * a.list_len + (g - before[l]));
    };
    int parity = 0;
    for (int item = blockIdx.x / n_blocks; item < n_runs; item += gridDim.x / n_blocks) {
        const int2 mine = run(item);
        if (threadIdx.x == 0) sh.end = a.n_rows;
        append_clear(sh);
        auto take = [&](int t) { atomicMax(&sh.win[__ldg(a.slots + t) & row_mask], t); };
        auto in_run = [&](int t) { return t < a.n_rows && append_page_of(a, __ldg(a.slots + t)) == mine.x; };
        if (!in_run(mine.y + threadIdx.x)) atomicMin(&sh.end, mine.y + static_cast<int>(threadIdx.x));
#pragma unroll 2
        for (int g = threadIdx.x; g < n_runs; g += kAppendThreads) {
            const int2 other = run(g);
            if (other.x != mine.x || other.y == mine.y) continue;
            if (other.y < mine.y) sh.earlier = 1;
            else
                for (int t = other.y; in_run(t); ++t) take(t);         // (seldom: the page comes up again)
        }
        __syncthreads();
        if (!sh.earlier) {                        // (alike in all blocks of the cluster)
            int t0 = mine.y;
            while (true) {                        // (once, unless slots are named twice)
                const int t = t0 + static_cast<int>(threadIdx.x), end = sh.end;
                if (t < end) take(t);
                __syncthreads();
                t0 += kAppendThreads;
                if (end < t0 || t0 >= a.n_rows) break;
                if (threadIdx.x == 0) sh.end = a.n_rows;
                __syncthreads();
                if (!in_run(t0 + threadIdx.x)) atomicMin(&sh.end, t0 + static_cast<int>(threadIdx.x));
                __syncthreads();
            }
            // this block's rows of the page
            const int r0 = rank * kAppendBlockRows, r1 = min(r0 + kAppendBlockRows, page_rows);
            const int r = r0 + static_cast<int>(threadIdx.x);
            if (r < r1 && sh.win[r] >= 0) sh.rows[atomicAdd(&sh.n_rows, 1)] = r;
            const float old = __ldcg(a.scales + mine.x);
            __syncthreads();
            const int slot = threadIdx.x / kAppendUnits, unit = threadIdx.x % kAppendUnits, n = sh.n_rows;
            auto source = [&](int i) { return __ldg(reinterpret_cast<const uint4*>(a.kv + static_cast<long long>(sh.win[sh.rows[i]]) * a.kv_stride) + unit); };
            uint32_t top = 0, finite;
#pragma unroll 4
            for (int i = slot; i < n; i += kAppendSide) top = max_bf16x2(top, source(i));
            top = finite = append_block_max(top, sh);
            if (top >= 0x7f80u) {
                finite = 0;
                __syncthreads();
                for (int i = slot; i < n; i += kAppendSide) finite = finite_max_bf16x2(finite, source(i));
                finite = append_block_max(finite, sh);
            }
            if (threadIdx.x == 0) *reinterpret_cast<uint2*>(page_max[parity]) = make_uint2(top, finite);
            cluster_sync_all();
            uint32_t tops[4], finites[4];         // (the first again where there are fewer blocks)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 other = ld_cluster_v4(map_to_cta(smem_u32(page_max[parity]), k < n_blocks ? k : 0));
                tops[k] = __float_as_uint(other.x);
                finites[k] = __float_as_uint(other.y);
            }
            top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
            finite = max(max(finites[0], finites[1]), max(finites[2], finites[3]));
            parity ^= 1;                          // (the next page's sync comes before this place is written again)
            const bool anew = sh.win[0] >= 0;
            const float wanted = exp2_int(scale_exp(finite << 16, kMinScaleExp)), scale = anew ? wanted : fmaxf(old, wanted);
            uint8_t* base = a.values + static_cast<size_t>(mine.x) * page_rows * kDQK;
            if (!anew && scale > old) append_rescale(sh, base, r0, r1, old / scale);
            if (threadIdx.x == 0 && rank == 0) a.scales[mine.x] = scale;
            const float inv = 1.f / scale;
#pragma unroll 4
            for (int i = slot; i < n; i += kAppendSide)
                *reinterpret_cast<uint2*>(base + static_cast<size_t>(sh.rows[i]) * kDQK + unit * 8) = append_cvt(source(i), inv, top < 0x7f80u);
        }
        __syncthreads();                          // (the next page's tables go to the same place)
    }
    cluster_sync_all();                           // (nobody leaves while another may read its maximum)
}

}  // namespace smla
