// A paged key/value cache: its pools, the page tables of a step, writing new
// tokens, and eviction by accumulated attention weight.
//
// Eviction keeps, for every sequence and key head, the `budget` slots with
// the largest keys (ties: the lower slot), where a slot's key is its score,
// or above every score for the newest `recent` positions and the first
// `sinks` ones. The kept rows below the budget stay where they are; the j-th
// kept slot past it moves into the j-th place that became free below it.
// Attention does not depend on the order of the slots, sources lie at or past
// the budget and destinations below it, so rows move in place, without a
// second copy of the cache and without a hazard. A slot's position is carried
// beside its score, since slots lose their order.
//
// Bytes: each score once, and twice the rows that move; after long prompts (4
// sequences x 8 heads of 65533 slots to 4096) 8.4 MB and 128 MB: the select
// takes 22.4 us, bound by the latency of its passes, the move 22.7 us = 5.6
// TB/s. After a few decoding steps (24 sequences x 8 heads, 1048 slots to 1024)
// one launch does both, in 12 us of the stream.
#include "operators.hpp"

#include <algorithm>
#include <sstream>
#include <stdexcept>
#include <unordered_set>

namespace porch::detail {

    namespace {

        void expect(bool ok, const std::string& message) {
            if (!ok) throw std::invalid_argument(message);
        }

        const char* append_source() {
            return R"PB(
typedef long long pb_i64;
// Thread: 8 values of one token's key and value. Bound by HBM: 4 B read and
// the cache's width written per value (65536 tokens x 8 heads x 128 into
// bfloat16: 117 us = 6.9 TB/s, into float32: 161 us = 6.7); a float32 value is rounded to nearest even
// bfloat16, the type that the cache holds.
static __device__ __forceinline__ pb_u32 pb_bf16_pair(float lo, float hi) {
    pb_u32 r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
extern "C" __global__ void __launch_bounds__(256) pb_cache_append(
    const float* k, const float* v, char* pk, char* pv, const pb_i64* rows, pb_i64 tokens,
    pb_i64 kt, pb_i64 kh, pb_i64 vt, pb_i64 vh) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_i64 n = tokens * PB_H * (PB_D / 8);
    const pb_i64 id = (pb_i64)blockIdx.x * 256 + threadIdx.x;
    if (id >= n) return;
    const int c = (int)(id % (PB_D / 8)) * 8;
    const pb_i64 th = id / (PB_D / 8);
    const int h = (int)(th % PB_H);
    const pb_i64 t = th / PB_H;
    const pb_i64 to = ((rows[t] / PB_PS * PB_H + h) * PB_PS + rows[t] % PB_PS) * PB_D + c;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const float* src = which ? v + t * vt + h * vh + c : k + t * kt + h * kh + c;
        float x[8];
#if PB_WIDE
        const float4 a = pb_ld4(src), b = pb_ld4(src + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
#else
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __ldg(src + e);
#endif
        char* dst = which ? pv : pk;
#if PB_BF16
        *reinterpret_cast<uint4*>(dst + to * 2) = make_uint4(pb_bf16_pair(x[0], x[1]), pb_bf16_pair(x[2], x[3]),
                                                             pb_bf16_pair(x[4], x[5]), pb_bf16_pair(x[6], x[7]));
#else
        *reinterpret_cast<float4*>(dst + to * 4) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(dst + to * 4 + 16) = make_float4(x[4], x[5], x[6], x[7]);
#endif
    }
}
)PB";
        }

        const char* evict_source() {
            return R"PB(
typedef long long pb_i64;
// An order-preserving map of floats to unsigned integers; NaN orders as -inf.
static __device__ __forceinline__ pb_u32 pb_order(float s) {
    if (!(s == s)) return 0x007fffffu;
    const pb_u32 u = __float_as_uint(s + 0.0f); // -0 becomes 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct pb_row {
    const float* scores; pb_i64 ns;    // this row's scores, and how many there are
    const float* places; pb_i64 np;
    int length; float newest, recent_from, sinks;
};
static __device__ __forceinline__ float pb_place(const pb_row& r, int i) {
    if (i < r.np) {
        const float p = r.places[i];
        if (p >= 0.0f) return p;
    }
    return r.newest - (float)(r.length - 1 - i);
}
static __device__ __forceinline__ float pb_score(const pb_row& r, int i) { return i < r.ns ? r.scores[i] : 0.0f; }
static __device__ __forceinline__ pb_u32 pb_key_of(const pb_row& r, int i, float score, float place) {
    const float p = place >= 0.0f ? place : r.newest - (float)(r.length - 1 - i); // NaN is no place
    return p > r.recent_from || p < r.sinks ? 0xffffffffu : pb_order(score);
}
static __device__ __forceinline__ pb_u32 pb_key(const pb_row& r, int i) {
    return pb_key_of(r, i, pb_score(r, i), i < r.np ? r.places[i] : -1.0f);
}

static __device__ __forceinline__ pb_row pb_row_of(const float* scores, const float* places, const int* lengths,
                                                   const int* newest, pb_i64 ns, pb_i64 np, int recent, int sinks,
                                                   pb_i64 row) {
    const int s = (int)(row / PB_H);
    pb_row r;
    r.scores = scores + row * ns;
    r.ns = ns;
    r.places = places + row * np;
    r.np = np;
    r.length = lengths[s];
    r.newest = (float)newest[s];
    r.recent_from = r.newest - (float)recent;
    r.sinks = (float)sinks;
    return r;
}
static __device__ __forceinline__ void pb_keep(const pb_row& r, float* out_scores, float* out_places, pb_i64 to, int i) {
    out_scores[to] = pb_score(r, i);
    out_places[to] = pb_place(r, i);
}

// Exclusive sums of two counts over the block's threads, and their totals.
static __device__ __forceinline__ int2 pb_block_scan(int2 v, int2* warps, int2& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockDim.x >> 5;
    int2 x = v;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const int a = __shfl_up_sync(0xffffffffu, x.x, m), b = __shfl_up_sync(0xffffffffu, x.y, m);
        if (lane >= m) { x.x += a; x.y += b; }
    }
    __syncthreads();
    if (lane == 31) warps[w] = x;
    __syncthreads();
    int2 before = make_int2(0, 0);
    total = before;
    int2 mine = lane < n ? warps[lane] : make_int2(0, 0);
    int2 sum = mine;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const int a = __shfl_up_sync(0xffffffffu, sum.x, m), b = __shfl_up_sync(0xffffffffu, sum.y, m);
        if (lane >= m) { sum.x += a; sum.y += b; }
    }
    total.x = __shfl_sync(0xffffffffu, sum.x, 31);
    total.y = __shfl_sync(0xffffffffu, sum.y, 31);
    before.x = __shfl_sync(0xffffffffu, sum.x - mine.x, w);
    before.y = __shfl_sync(0xffffffffu, sum.y - mine.y, w);
    return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// The digit of the `want`-th largest key among 256 counted bins, how many
// keys of its bin are wanted, and whether that is all of them. One warp.
static __device__ __forceinline__ void pb_pick(const int* bins, int want, int* chosen) {
    const int lane = threadIdx.x & 31;
    int own[8], sum = 0; // bins 255 - 8 lane, downwards
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += own[j] = bins[255 - 8 * lane - j];
    int upto = sum;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const int a = __shfl_up_sync(0xffffffffu, upto, m);
        if (lane >= m) upto += a;
    }
    int left = want - (upto - sum);
    if (left > 0 && left <= sum) {
        int j = 0;
        while (own[j] < left) left -= own[j++];
        chosen[0] = 255 - 8 * lane - j;
        chosen[1] = left;
        chosen[2] = own[j] == left;
    }
}

// Up to PB_MOVES pairs of one row: late slot and free place, one a lane.
struct pb_pairs { int from, to, count; };
static __device__ __forceinline__ pb_pairs pb_list(const int* holes, const int* lates, const int* counts, pb_i64 row,
                                                   int group, int pairs) {
    pb_pairs p = {0, 0, 0};
    const int lane = threadIdx.x & 31, j = group * PB_MOVES;
    if (lane < PB_MOVES && j + lane < pairs) { // read beside the count; what lies past it is not used
        p.from = lates[row * pairs + j + lane];
        p.to = holes[row * pairs + j + lane];
    }
    p.count = min(PB_MOVES, counts[row] - j);
    if (lane >= p.count) p.from = p.to = 0;
    return p;
}

// Moves the pairs' rows, keys and values, with their scores and positions: one
// warp, all loads before the first store, so that it has as many bytes on the
// way as PB_MOVES rows. Sources lie at or past the budget, destinations below.
static __device__ __forceinline__ void pb_move(const pb_pairs& p, const pb_row& r, char* pk, char* pv, const int* tables,
                                               float* out_scores, float* out_places, pb_i64 row, int width, int budget) {
    const int lane = threadIdx.x & 31, h = (int)(row % PB_H);
    const int* table = tables + row / PB_H * width;
    // Lane m finds where pair m's rows lie; all lanes move them.
    pb_i64 from = 0, to = 0;
    if (lane < p.count) {
        from = (((pb_i64)__ldg(table + p.from / PB_PS) * PB_H + h) * PB_PS + p.from % PB_PS) * PB_ROW;
        to = (((pb_i64)__ldg(table + p.to / PB_PS) * PB_H + h) * PB_PS + p.to % PB_PS) * PB_ROW;
    }
    // 16 bytes a lane: chunk c of the 2 * PB_ROW bytes of a slot, keys first.
    uint4 v[PB_MOVES][PB_CHUNKS];
#pragma unroll
    for (int m = 0; m < PB_MOVES; ++m) {
        const pb_i64 a = __shfl_sync(0xffffffffu, from, m);
#pragma unroll
        for (int c = 0; c < PB_CHUNKS; ++c) {
            const int at = (c * 32 + lane) * 16;
            if (m < p.count && at < 2 * PB_ROW)
                v[m][c] = __ldcs(reinterpret_cast<const uint4*>((at < PB_ROW ? pk + at : pv + at - PB_ROW) + a));
        }
    }
    if (lane < p.count) pb_keep(r, out_scores, out_places, row * budget + p.to, p.from);
#pragma unroll
    for (int m = 0; m < PB_MOVES; ++m) {
        const pb_i64 b = __shfl_sync(0xffffffffu, to, m);
#pragma unroll
        for (int c = 0; c < PB_CHUNKS; ++c) {
            const int at = (c * 32 + lane) * 16;
            if (m < p.count && at < 2 * PB_ROW)
                __stcs(reinterpret_cast<uint4*>((at < PB_ROW ? pk + at : pv + at - PB_ROW) + b), v[m][c]);
        }
    }
}

#ifdef PB_CLUSTER
static __device__ __forceinline__ pb_u32 pb_rank() {
    pb_u32 r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
static __device__ __forceinline__ void pb_cluster_sync() {
#if PB_CLUSTER > 1
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
#else
    __syncthreads();
#endif
}
// An int of CTA `rank` of the cluster.
static __device__ __forceinline__ int pb_peer(const int* p, pb_u32 rank) {
    int v;
    pb_u32 a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((pb_u32)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// Sums of two of the counts that CTAs of lower rank left in `totals`.
static __device__ __forceinline__ int2 pb_before(const int* totals, pb_u32 rank, int2* sums) {
#if PB_CLUSTER > 1
    if (threadIdx.x < 32) {
        int2 v = make_int2(0, 0);
        if (threadIdx.x < rank) v = make_int2(pb_peer(totals, threadIdx.x), pb_peer(totals + 1, threadIdx.x));
#pragma unroll
        for (int m = 4; m > 0; m /= 2) {
            v.x += __shfl_down_sync(0xffffffffu, v.x, m);
            v.y += __shfl_down_sync(0xffffffffu, v.y, m);
        }
        if (threadIdx.x == 0) *sums = v;
    }
    __syncthreads();
    return *sums;
#else
    return make_int2(0, 0);
#endif
}

#ifndef PB_LONG
// One cluster per sequence and key head. Each CTA holds the keys of a run of
// slots; a thread owns PB_KPT consecutive ones, handed over through shared
// memory (an odd stride apart, so that threads use distinct banks), and the
// row is read once:
//  1. radix select of the budget-th largest key, 8 bits a pass, the counts
//     summed over the cluster through distributed shared memory; it ends as
//     soon as a bin is wanted whole;
//  2. exclusive sums over the slots' order rank ties, free places and late
//     slots. The j-th late slot goes to the j-th free place;
//  3. where they are few (`fused`) its warps move them, which saves a launch.
// What bounds it: the latency of the passes (two barriers each), not bytes.
extern "C" __global__ void __launch_bounds__(PB_THREADS, PB_THREADS < 1024 ? 2 : 1) pb_evict_select(
    const float* scores, const float* places, const int* lengths, const int* newest, float* out_scores,
    float* out_places, int* holes, int* lates, int* counts, pb_i64 ns, pb_i64 np, int budget, int recent, int sinks,
    int pairs, char* pk, char* pv, const int* tables, int width, int fused) {
    constexpr int threads = PB_THREADS, run = PB_THREADS * PB_KPT, stride = PB_KPT | 1;
    extern __shared__ pb_u32 keys[];
    __shared__ int hist[2][256], bins[256], chosen[3], totals[4];
    __shared__ int2 warps[32], before;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_i64 row = blockIdx.x / PB_CLUSTER;
    const pb_u32 rank = PB_CLUSTER > 1 ? pb_rank() : 0;
    const pb_row r = pb_row_of(scores, places, lengths, newest, ns, np, recent, sinks, row);
    const int first = rank * run;
    // Nothing is kept past the length; the budget may reach past the cluster's slots.
    for (int i = max(r.length, first) + threadIdx.x; i < (rank == PB_CLUSTER - 1 ? budget : min(first + run, budget)); i += threads) {
        out_scores[row * budget + i] = 0.0f;
        out_places[row * budget + i] = -1.0f;
    }
    if (r.length <= budget) { // the same in every CTA of the cluster
        for (int i = first + threadIdx.x; i < min(first + run, r.length); i += threads)
            pb_keep(r, out_scores, out_places, row * budget + i, i);
        if (rank == 0 && threadIdx.x == 0) counts[row] = 0;
        return;
    }
    const int n = min(run, r.length - first); // may be negative
    constexpr int batch = PB_KPT < 16 ? PB_KPT : 16; // loads on the way at once
#pragma unroll 1
    for (int q = 0; q < PB_KPT; q += batch) {
        float score[batch], place[batch];
#pragma unroll
        for (int j = 0; j < batch; ++j) { // every load before the first use
            const int i = first + (q + j) * threads + threadIdx.x;
            score[j] = i < r.length && i < r.ns ? r.scores[i] : 0.0f;
            place[j] = i < r.length && i < r.np ? r.places[i] : -1.0f;
        }
#pragma unroll
        for (int j = 0; j < batch; ++j) {
            const int i = (q + j) * threads + threadIdx.x;
            keys[i / PB_KPT * stride + i % PB_KPT] = pb_key_of(r, first + i, score[j], place[j]);
        }
    }
    pb_u32* own = keys + threadIdx.x * stride;
    const int mine = max(0, min(PB_KPT, n - (int)threadIdx.x * PB_KPT));

    pb_u32 limit = 0; // the bits of the threshold so far
    int want = budget;
    bool whole = false;
    for (int i = threadIdx.x; i < 256; i += threads) hist[0][i] = 0;
    __syncthreads();
    for (int pass = 0; pass < 4 && !whole; ++pass) {
        const int shift = 24 - 8 * pass;
        int* h = hist[pass & 1];
        for (int j = 0; j < mine; ++j) {
            const pb_u32 key = own[j];
            if (pass == 0 || ((key ^ limit) >> (shift + 8)) == 0) atomicAdd(&h[(key >> shift) & 255u], 1);
        }
        pb_cluster_sync();
        for (int i = threadIdx.x; i < 256; i += threads) {
            int sum = 0;
#pragma unroll
            for (int c = 0; c < PB_CLUSTER; ++c) sum += PB_CLUSTER > 1 ? pb_peer(h + i, c) : h[i];
            bins[i] = sum;
            hist[(pass & 1) ^ 1][i] = 0; // every CTA has read it: it was before this barrier
        }
        __syncthreads();
        if (threadIdx.x < 32) pb_pick(bins, want, chosen);
        __syncthreads();
        limit |= (pb_u32)chosen[0] << shift;
        want = chosen[1];
        whole = chosen[2];
    }
    // Kept: keys above the limit, and of those equal to it the first `want`
    // (all of them where a bin was wanted whole: then the limit's low bits are 0).
    int2 total;
    int ties = 0;
    if (!whole) {
        int count = 0;
        for (int j = 0; j < mine; ++j) count += own[j] == limit;
        ties = pb_block_scan(make_int2(count, 0), warps, total).x;
        if (threadIdx.x == 0) totals[0] = total.x;
        pb_cluster_sync();
        ties += pb_before(totals, rank, &before).x;
    }
    pb_u64 kept = 0; // up to 64 slots a thread
    int2 count = make_int2(0, 0); // free places, late slots
    int seen = ties;
    const int slot0 = first + threadIdx.x * PB_KPT;
    for (int j = 0; j < mine; ++j) {
        const pb_u32 key = own[j];
        const bool keep = whole ? key >= limit : key > limit || (key == limit && seen++ < want);
        kept |= (pb_u64)keep << j;
        const bool low = slot0 + j < budget;
        count.x += low && !keep;
        count.y += !low && keep;
    }
    int2 at = pb_block_scan(count, warps, total);
    if (threadIdx.x == 0) { totals[2] = total.x; totals[3] = total.y; }
    pb_cluster_sync();
    const int2 earlier = pb_before(totals + 2, rank, &before);
    at.x += earlier.x;
    at.y += earlier.y;
    for (int j = 0; j < mine; ++j) {
        const int i = slot0 + j;
        const bool keep = kept >> j & 1u;
        if (i < budget && !keep) holes[row * pairs + at.x++] = i;
        if (i >= budget && keep) lates[row * pairs + at.y++] = i;
        own[j] = keep;
    }
    __syncthreads();
    // Slots that stay where they are: their scores and positions, four on the way.
    const int stay = min(n, budget - first);
    for (int base = threadIdx.x; base < stay; base += 4 * threads) {
        float score[4], place[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + j * threads;
            const bool keep = i < stay && keys[i / PB_KPT * stride + i % PB_KPT];
            score[j] = keep ? pb_score(r, first + i) : 0.0f;
            place[j] = keep ? pb_place(r, first + i) : -1.0f; // a position is not negative
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (place[j] >= 0.0f) {
                out_scores[row * budget + first + base + j * threads] = score[j];
                out_places[row * budget + first + base + j * threads] = place[j];
            }
    }
    if (rank == PB_CLUSTER - 1 && threadIdx.x == threads - 1) counts[row] = at.y;
    // The row's lists are complete, and nobody leaves while its shared memory is read.
    pb_cluster_sync();
    if (fused) {
        const int groups = (pairs + PB_MOVES - 1) / PB_MOVES;
        for (int g = rank * (threads / 32) + (threadIdx.x >> 5); g < groups; g += PB_CLUSTER * (threads / 32)) {
            const pb_pairs p = pb_list(holes, lates, counts, row, g, pairs);
            if (p.count <= 0) break;
            pb_move(p, r, pk, pv, tables, out_scores, out_places, row, width, budget);
        }
    }
}
#endif
#endif

#if defined(PB_CLUSTER) && defined(PB_LONG)
// The same for rows whose keys do not fit a cluster's shared memory: each CTA
// reads its run of slots again, 4096 at a time, in every pass of the select,
// once to count what it keeps, and once to write. One row of 420000
// slots: 1137 us with one CTA, 104 with 8 (of 390000, held: 43).
extern "C" __global__ void __launch_bounds__(1024) pb_evict_select_long(
    const float* scores, const float* places, const int* lengths, const int* newest, float* out_scores,
    float* out_places, int* holes, int* lates, int* counts, pb_i64 ns, pb_i64 np, int budget, int recent, int sinks,
    int pairs) {
    constexpr int round = 4096;
    __shared__ int hist[2][256], bins[256], chosen[3], totals[4];
    __shared__ int2 warps[32], before[2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_i64 row = blockIdx.x / PB_CLUSTER;
    const int rank = (int)pb_rank();
    const pb_row r = pb_row_of(scores, places, lengths, newest, ns, np, recent, sinks, row);
    for (pb_i64 i = (pb_i64)r.length + rank * 1024 + threadIdx.x; i < budget; i += PB_CLUSTER * 1024) {
        out_scores[row * budget + i] = 0.0f;
        out_places[row * budget + i] = -1.0f;
    }
    if (r.length <= budget) { // the same in every CTA of the cluster
        for (int i = rank * 1024 + threadIdx.x; i < r.length; i += PB_CLUSTER * 1024)
            pb_keep(r, out_scores, out_places, row * budget + i, i);
        if (rank == 0 && threadIdx.x == 0) counts[row] = 0;
        return;
    }
    const int run = (r.length + PB_CLUSTER * round - 1) / (PB_CLUSTER * round) * round;
    const int first = (int)min((pb_i64)rank * run, (pb_i64)r.length), last = (int)min((pb_i64)first + run, (pb_i64)r.length);
    // This thread's four slots of the round at `base`, every load before the first use.
    auto load = [&](int base, pb_u32* key) {
        float score[4], place[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + threadIdx.x * 4 + j;
            score[j] = i < last && i < r.ns ? r.scores[i] : 0.0f;
            place[j] = i < last && i < r.np ? r.places[i] : -1.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) key[j] = pb_key_of(r, base + threadIdx.x * 4 + j, score[j], place[j]);
    };

    pb_u32 limit = 0;
    int want = budget;
    bool whole = false;
    for (int i = threadIdx.x; i < 256; i += 1024) hist[0][i] = 0;
    __syncthreads();
    for (int pass = 0; pass < 4 && !whole; ++pass) {
        const int shift = 24 - 8 * pass;
        int* h = hist[pass & 1];
        for (int base = first; base < last; base += round) {
            pb_u32 key[4];
            load(base, key);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (base + (int)threadIdx.x * 4 + j < last && (pass == 0 || ((key[j] ^ limit) >> (shift + 8)) == 0))
                    atomicAdd(&h[(key[j] >> shift) & 255u], 1);
        }
        pb_cluster_sync();
        for (int i = threadIdx.x; i < 256; i += 1024) {
            int sum = 0;
#pragma unroll
            for (int c = 0; c < PB_CLUSTER; ++c) sum += pb_peer(h + i, c);
            bins[i] = sum;
            hist[(pass & 1) ^ 1][i] = 0; // every CTA has read it: it was before this barrier
        }
        __syncthreads();
        if (threadIdx.x < 32) pb_pick(bins, want, chosen);
        __syncthreads();
        limit |= (pb_u32)chosen[0] << shift;
        want = chosen[1];
        whole = chosen[2];
    }

    // Keys equal to the limit and keys above it, below the budget and past it.
    int2 equal = make_int2(0, 0), above = make_int2(0, 0), total;
    for (int base = first; base < last; base += round) {
        pb_u32 key[4];
        load(base, key);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + threadIdx.x * 4 + j;
            if (i >= last) continue;
            const bool over = whole ? key[j] >= limit : key[j] > limit, same = !whole && key[j] == limit;
            equal.x += same && i < budget;
            equal.y += same && i >= budget;
            above.x += over && i < budget;
            above.y += over && i >= budget;
        }
    }
    (void)pb_block_scan(equal, warps, total);
    if (threadIdx.x == 0) { totals[0] = total.x; totals[1] = total.y; }
    (void)pb_block_scan(above, warps, total);
    if (threadIdx.x == 0) { totals[2] = total.x; totals[3] = total.y; }
    pb_cluster_sync();
    if (threadIdx.x < 32) {
        // Lane c: what CTA c keeps, given the ties of those before it.
        const int c = threadIdx.x;
        int t[4] = {0, 0, 0, 0};
        if (c < PB_CLUSTER)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = pb_peer(totals + j, c);
        int ties = t[0] + t[1];
#pragma unroll
        for (int m = 1; m < PB_CLUSTER; m *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, ties, m);
            if (c >= m) ties += v;
        }
        ties -= t[0] + t[1];
        const int kept = max(0, min(want - ties, t[0] + t[1])), low = min(kept, t[0]);
        const pb_i64 from = (pb_i64)c * run;
        const int slots = (int)max((pb_i64)0, min((pb_i64)budget, min(from + run, (pb_i64)r.length)) - from);
        int2 sum = c < rank ? make_int2(slots - t[2] - low, t[3] + kept - low) : make_int2(0, 0);
#pragma unroll
        for (int m = 4; m > 0; m /= 2) {
            sum.x += __shfl_down_sync(0xffffffffu, sum.x, m);
            sum.y += __shfl_down_sync(0xffffffffu, sum.y, m);
        }
        if (c == 0) before[0] = sum;
        if (c == rank) before[1] = make_int2(ties, 0);
    }
    __syncthreads();
    int2 at = before[0]; // free places and late slots so far
    int ties = before[1].x;
    for (int base = first; base < last; base += round) {
        pb_u32 key[4];
        load(base, key);
        const int i0 = base + threadIdx.x * 4;
        int seen = ties;
        if (!whole) {
            int same = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) same += i0 + j < last && key[j] == limit;
            seen += pb_block_scan(make_int2(same, 0), warps, total).x;
            ties += total.x;
        }
        int2 count = make_int2(0, 0);
        int kept = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j >= last) continue;
            const bool keep = whole ? key[j] >= limit : key[j] > limit || (key[j] == limit && seen++ < want);
            kept |= keep << j;
            count.x += i0 + j < budget && !keep;
            count.y += i0 + j >= budget && keep;
        }
        int2 mine = pb_block_scan(count, warps, total);
        mine.x += at.x;
        mine.y += at.y;
        at.x += total.x;
        at.y += total.y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j;
            if (i >= last) continue;
            const bool keep = kept >> j & 1;
            if (i < budget && !keep) holes[row * pairs + mine.x++] = i;
            if (i < budget && keep) pb_keep(r, out_scores, out_places, row * budget + i, i);
            if (i >= budget && keep) lates[row * pairs + mine.y++] = i;
        }
    }
    if (rank == PB_CLUSTER - 1 && threadIdx.x == 0) counts[row] = at.y;
    pb_cluster_sync(); // nobody leaves while its shared memory is read
}
#endif

#ifndef PB_CLUSTER
extern "C" __global__ void __launch_bounds__(256) pb_evict_move(
    char* pk, char* pv, const int* tables, const float* scores, const float* places, const int* lengths,
    const int* newest, float* out_scores, float* out_places, const int* holes, const int* lates, const int* counts,
    pb_i64 ns, pb_i64 np, int width, int budget, int pairs, pb_u32 blocks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Blocks of 8 warps, `blocks` of them for each row.
    const pb_i64 row = blockIdx.x / blocks;
    const pb_pairs p = pb_list(holes, lates, counts, row, (blockIdx.x % blocks) * 8 + (threadIdx.x >> 5), pairs);
    if (p.count <= 0) return;
    const pb_row r = pb_row_of(scores, places, lengths, newest, ns, np, 0, 0, row);
    pb_move(p, r, pk, pv, tables, out_scores, out_places, row, width, budget);
}
#endif
)PB";
        }

        // How the select shares out a row of `longest` slots.
        struct select_shape {
            int cluster = 0, threads = 0, per_thread = 0;
            bool held = true; // false: the long form, which reads the row again
            uint32_t smem() const { return held ? static_cast<uint32_t>(threads * (per_thread | 1) * 4) : 0; }
        };
        select_shape shape_for(int64_t longest, int64_t rows, int sms) {
            static constexpr int kShapes[][2] = {{256, 4}, {256, 8}, {512, 8}, {512, 16}, {1024, 16}, {1024, 32}, {1024, 48}};
            select_shape r;
            // More CTAs for each row as long as every CTA has an SM of its own and
            // a few thousand slots (32 rows of 65533 slots: 22.4 us with 4 CTAs of
            // 1024 threads each, 23.5 with 8 of 512, two of an SM, 31.9 with 2);
            // more still where the keys need the room.
            int64_t c = 1;
            while (c < 8 && rows * c * 2 <= sms && longest >= 4096 * c) c *= 2;
            for (; c <= 8; c *= 2)
                for (const auto& [threads, per_thread] : kShapes)
                    if (int64_t{threads} * per_thread * c >= longest) {
                        r.cluster = static_cast<int>(c);
                        r.threads = threads;
                        r.per_thread = per_thread;
                        return r;
                    }
            r = {8, 1024, 4, false};
            return r;
        }

        // Rows with at most so many late slots move them in the select, which
        // saves a launch (24 of 1048 slots: 22.0 us a call with two, 19.5 so). Of
        // thousands of slots the move alone keeps more SMs busy (48.4 us, 52.3 so).
        constexpr int kFewPairs = 128;

        // Pairs that a warp moves: 2 KB on the way, more where one pair is larger.
        // 64 MB of pairs take 24.8 us with 1 KB, 22.7 with 2 and 22.0 with 4,
        // which costs the select, where it moves few pairs itself, its registers.
        int moves_of(const kv_cache& c) { return std::max<int>(1, 4 / static_cast<int>((2 * c.dim * c.width() + 511) / 512)); }

        std::string defines(const kv_cache& c, bool wide, const select_shape& f = {}) {
            std::ostringstream os;
            os << "#define PB_H " << c.heads << "\n#define PB_D " << c.dim << "\n#define PB_PS " << c.page_size
               << "\n#define PB_ROW " << c.dim * c.width() << "\n#define PB_BF16 " << (c.type == cache_type::bf16 ? 1 : 0)
               << "\n#define PB_WIDE " << (wide ? 1 : 0) << "\n#define PB_MOVES " << moves_of(c)
               << "\n#define PB_CHUNKS " << (2 * c.dim * c.width() + 511) / 512 << "\n";
            if (f.cluster != 0)
                os << "#define PB_CLUSTER " << f.cluster << "\n#define PB_THREADS " << f.threads << "\n#define PB_KPT "
                   << f.per_thread << "\n" << (f.held ? "" : "#define PB_LONG 1\n");
            return os.str();
        }

        const char kAppend[] = "pb_cache_append";
        const char kSelect[] = "pb_evict_select";
        const char kSelectLong[] = "pb_evict_select_long";
        const char kMove[] = "pb_evict_move";

        op_kernel& kernel_of(const char* name, const kv_cache& c, bool wide = true, const select_shape& f = {}) {
            const op_key key{reinterpret_cast<int64_t>(name), c.heads, c.dim, c.page_size, static_cast<int64_t>(c.type),
                             wide, f.cluster, f.threads, f.per_thread, f.held};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = name;
                k.source = std::string{kernel_prelude()} + defines(c, wide, f) +
                           (name == kAppend ? append_source() : evict_source());
                k.smem = f.smem();
            });
        }

    } // namespace

    std::shared_ptr<kv_cache> make_cache(int64_t pages, int64_t page_size, int64_t heads, int64_t dim,
                                         cache_type type, int device) {
        expect(type == cache_type::f32 || type == cache_type::bf16, "cache: type must be float32 or bfloat16");
        expect(pages >= 1 && pages <= (int64_t{1} << 30), "cache: pages must be 1 to 2^30");
        expect(page_size >= 8 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
               "cache: page_size must be a power of two from 8 to 256");
        expect(heads >= 1 && heads <= 1024, "cache: kv_heads must be 1 to 1024");
        expect(dim >= 8 && dim <= 256 && dim % 8 == 0, "cache: head_dim must be a multiple of 8 up to 256");
        // Rows are counted in 31 bits by the tile loads.
        expect(pages * heads * page_size < (int64_t{1} << 31), "cache: pages x kv_heads x page_size must be below 2^31");
        int ndev = 0;
        check(pbrt_device_count(&ndev));
        auto c = std::make_shared<kv_cache>();
        c->pages = pages;
        c->page_size = page_size;
        c->heads = heads;
        c->dim = dim;
        c->type = type;
        c->device = checked_ordinal(device, ndev);
        const size_t bytes = static_cast<size_t>(pages * heads * page_size * dim) * static_cast<size_t>(c->width());
        auto stream = current_stream(c->device);
        c->k = allocate(c->device, bytes, stream);
        c->v = allocate(c->device, bytes, stream);
        const uint64_t dims[2] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(pages * heads * page_size)};
        const uint64_t strides[1] = {static_cast<uint64_t>(dim * c->width())};
        const uint32_t box[2] = {static_cast<uint32_t>(128 / c->width()), static_cast<uint32_t>(std::min<int64_t>(64, page_size))};
        const uint32_t ones[2] = {1, 1};
        // bfloat16 or float32, 128-byte swizzle, 256-byte L2 promotion, zeros past the head size.
        for (auto [m, p] : {std::pair{&c->map_k, &c->k}, std::pair{&c->map_v, &c->v}})
            check(pbrt_tensor_map_encode_tiled(m->bytes, type == cache_type::bf16 ? 9 : 7, 2, address(*p), dims, strides,
                                               box, ones, 0, 3, 3, 0));
        return c;
    }

    pbrt_stream cache_ordered(kv_cache& c) {
        auto stream = current_stream(c.device);
        std::scoped_lock lock{c.order};
        order_read(*cuda_jit::buffer_access::state(c.k), stream);
        order_read(*cuda_jit::buffer_access::state(c.v), stream);
        return stream->stream;
    }

    std::shared_ptr<kv_batch> make_batch(std::shared_ptr<kv_cache> cache, const int32_t* tables, size_t sequences,
                                         size_t width, const int64_t* lengths, const int64_t* appended,
                                         const int64_t* newest) {
        const int64_t page = cache->page_size;
        expect(sequences >= 1 && sequences <= 65535, "cache batch: 1 to 65535 sequences");
        auto b = std::make_shared<kv_batch>();
        b->cache = cache;
        b->lengths.assign(lengths, lengths + sequences);
        std::vector<char> used(static_cast<size_t>(cache->pages), 0);
        std::vector<int64_t> rows;
        for (size_t s = 0; s < sequences; ++s) {
            const int64_t n = lengths[s];
            const std::string at = "cache batch: sequence " + std::to_string(s) + ": ";
            expect(n >= 0 && n < (int64_t{1} << 30), at + "length must be 0 to 2^30");
            const int64_t pages = (n + page - 1) / page;
            expect(pages <= static_cast<int64_t>(width), at + "its page table is too short for its length");
            for (int64_t j = 0; j < pages; ++j) {
                const int32_t p = tables[s * width + static_cast<size_t>(j)];
                if (p < 0 || p >= cache->pages)
                    throw std::out_of_range(at + "page " + std::to_string(p) + " is not one of the cache's");
                if (used[static_cast<size_t>(p)]++) {
                    used[static_cast<size_t>(p)] = 1;
                    b->shared_pages = true;
                }
            }
            const int64_t fresh = appended != nullptr ? appended[s] : std::min<int64_t>(1, n);
            expect(fresh >= 0 && fresh <= n, at + "new tokens must be 0 to its length");
            for (int64_t i = n - fresh; i < n; ++i)
                rows.push_back(int64_t{tables[s * width + static_cast<size_t>(i / page)]} * page + i % page);
            const int64_t last = newest != nullptr ? newest[s] : std::max<int64_t>(0, n - 1);
            expect(last >= 0 && last < (int64_t{1} << 24), at + "newest position must be 0 to 2^24 (float32 counts them exactly)");
            expect(newest == nullptr || n == 0 || last >= n - 1, at + "newest position must be at least its length - 1");
            b->newest.push_back(last);
            b->longest = std::max(b->longest, n);
            b->table_width = std::max(b->table_width, pages);
        }
        if (b->shared_pages) {
            std::unordered_set<int64_t> distinct(rows.begin(), rows.end());
            expect(distinct.size() == rows.size(), "cache batch: two new tokens go to the same row");
        }
        b->tokens = static_cast<int64_t>(rows.size());
        b->table_width = std::max<int64_t>(1, b->table_width);

        // One upload: lengths, newest, tables, rows (8-byte aligned).
        std::vector<int32_t> host;
        host.reserve(sequences * (2 + static_cast<size_t>(b->table_width)) + 2 * rows.size() + 1);
        for (int64_t n : b->lengths) host.push_back(static_cast<int32_t>(n));
        for (int64_t n : b->newest) host.push_back(static_cast<int32_t>(n));
        const size_t tables_from = host.size();
        for (size_t s = 0; s < sequences; ++s)
            for (int64_t j = 0; j < b->table_width; ++j)
                host.push_back(j * page < lengths[s] ? tables[s * width + static_cast<size_t>(j)] : 0);
        if (host.size() % 2 != 0) host.push_back(0);
        const size_t rows_from = host.size();
        for (int64_t r : rows) {
            host.push_back(static_cast<int32_t>(static_cast<uint64_t>(r) & 0xffffffffu));
            host.push_back(static_cast<int32_t>(static_cast<uint64_t>(r) >> 32));
        }
        // On the upload stream, so that waiting for the copy does not wait
        // for the step that is still running.
        auto stream = upload_stream(cache->device);
        b->data = allocate(cache->device, host.size() * sizeof(int32_t), stream);
        const uint64_t at = address(b->data);
        check(pbrt_memcpy_h2d_async(cache->device, at, host.data(), host.size() * sizeof(int32_t), stream->stream));
        check(pbrt_stream_synchronize(cache->device, stream->stream));
        b->lengths_at = at;
        b->newest_at = at + sequences * sizeof(int32_t);
        b->tables_at = at + tables_from * sizeof(int32_t);
        b->rows_at = at + rows_from * sizeof(int32_t);
        b->plans->hint = cache->hint;
        prepare_plan(*b);
        return b;
    }

    std::shared_ptr<kv_batch> batch_on(const kv_batch& batch, std::shared_ptr<kv_cache> cache) {
        const kv_cache &a = *batch.cache, &b = *cache;
        expect(a.pages == b.pages && a.page_size == b.page_size && a.heads == b.heads && a.dim == b.dim &&
                   a.type == b.type && a.device == b.device,
               "cache batch: the other cache has another shape, type or device");
        auto r = std::make_shared<kv_batch>(batch);
        r->cache = std::move(cache);
        return r;
    }

    void cache_append(kv_batch& batch, const tensor& k, const tensor& v) {
        kv_cache& c = *batch.cache;
        const std::vector<index_t> want{batch.tokens, c.heads, c.dim};
        expect(shape_of(k) == want && shape_of(v) == want,
               "cache_append: k and v must be [new tokens, kv_heads, head_dim] of the batch");
        const int device = device_of(k, "cache_append");
        expect(device == c.device && device_of(v, "cache_append") == c.device, "cache_append: operands must live on the cache's device");
        if (batch.tokens == 0) return;
        auto stream = current_stream(device);
        op_operand xk = operand(k, stream, true), xv = operand(v, stream, true);
        const bool wide = std::min(vector_width(xk), vector_width(xv)) == 4;
        op_kernel& kernel = kernel_of(kAppend, c, wide);
        (void)kernel.on(device);
        uint64_t pk = address(c.k), pv = address(c.v);
        const int64_t blocks = (batch.tokens * c.heads * (c.dim / 8) + 255) / 256;
        expect(blocks <= 0x7fffffff, "cache_append: too many new tokens");
        void* params[] = {&xk.ptr,        &xv.ptr,        &pk,            &pv,            &batch.rows_at,
                          &batch.tokens,  &xk.strides[0], &xk.strides[1], &xv.strides[0], &xv.strides[1]};
        order_read(*cuda_jit::buffer_access::state(batch.data), stream);
        std::scoped_lock lock{c.order};
        order_write(*cuda_jit::buffer_access::state(c.k), stream);
        order_write(*cuda_jit::buffer_access::state(c.v), stream);
        op_launch(kernel, device, stream, {static_cast<uint32_t>(blocks), 1, 1}, 256, params);
    }

    std::array<tensor, 2> cache_evict(kv_batch& batch, const tensor& scores, const tensor* positions,
                                      int64_t budget, int64_t recent, int64_t sinks) {
        kv_cache& c = *batch.cache;
        const int64_t n = batch.sequences();
        auto rows_of = [&](const tensor& t, const char* what) {
            const auto s = shape_of(t);
            expect(s.size() == 3 && s[0] == n && s[1] == c.heads,
                   std::string{"cache_evict: "} + what + " must be [sequences, kv_heads, slots]");
            return s[2];
        };
        const int64_t ns = rows_of(scores, "scores");
        const int64_t np = positions != nullptr ? rows_of(*positions, "positions") : 0;
        expect(budget >= 1 && budget < (int64_t{1} << 30), "cache_evict: budget must be 1 to 2^30");
        expect(recent >= 0 && sinks >= 0 && recent <= budget && sinks <= budget - recent,
               "cache_evict: recent and sinks must not be negative, and together at most the budget");
        expect(!batch.shared_pages, "cache_evict: a page of the batch serves more than one place, so its rows cannot move");
        const int device = device_of(scores, "cache_evict");
        expect(device == c.device && (positions == nullptr || device_of(*positions, "cache_evict") == device),
               "cache_evict: operands must live on the cache's device");
        auto stream = current_stream(device);
        op_operand xs = operand(scores, stream, false), xp;
        if (positions != nullptr) xp = operand(*positions, stream, false);
        const std::vector<index_t> out{n, c.heads, budget};
        op_result os = new_result(out, device, stream), op = new_result(out, device, stream);
        int64_t rows = n * c.heads;
        // No row has more late slots than it has places, or slots past the budget.
        int pairs = static_cast<int>(std::max<int64_t>(1, std::min(budget, batch.longest - budget)));
        const size_t list = static_cast<size_t>(rows) * static_cast<size_t>(pairs);
        auto scratch = allocate(device, (2 * list + static_cast<size_t>(rows)) * sizeof(int32_t), stream);
        uint64_t holes = address(scratch), lates = holes + list * 4, counts = lates + list * 4;
        order_read(*cuda_jit::buffer_access::state(batch.data), stream);
        int b = static_cast<int>(budget), rc = static_cast<int>(recent), sk = static_cast<int>(sinks);
        int width = static_cast<int>(batch.table_width);
        int64_t nsv = ns, npv = np;
        select_shape f = shape_for(batch.longest, rows, sm_count(device));
        const bool moves = batch.longest > budget;
        uint64_t pk = address(c.k), pv = address(c.v);
        int fused = moves && f.held && pairs <= kFewPairs;
        op_kernel& select = kernel_of(f.held ? kSelect : kSelectLong, c, true, f);
        op_kernel* move = moves && !fused ? &kernel_of(kMove, c) : nullptr;
        uint32_t per_row = static_cast<uint32_t>((pairs + 8 * moves_of(c) - 1) / (8 * moves_of(c)));
        const int64_t blocks = rows * per_row; // of the move
        expect(move == nullptr || blocks <= 0x7fffffff, "cache_evict: too many rows");
        (void)select.on(device);
        if (move != nullptr) (void)move->on(device);
        void* sparams[] = {&xs.ptr, &xp.ptr, &batch.lengths_at, &batch.newest_at, &os.ptr, &op.ptr, &holes,
                           &lates,  &counts, &nsv,              &npv,             &b,      &rc,     &sk,
                           &pairs,  &pk,     &pv,               &batch.tables_at, &width,  &fused};
        void* mparams[] = {&pk,     &pv,    &batch.tables_at, &xs.ptr, &xp.ptr, &batch.lengths_at, &batch.newest_at,
                           &os.ptr, &op.ptr, &holes,          &lates,  &counts, &nsv,              &npv,
                           &width, &b,      &pairs,           &per_row};
        {
            std::scoped_lock lock{c.order};
            if (moves) {
                order_write(*cuda_jit::buffer_access::state(c.k), stream);
                order_write(*cuda_jit::buffer_access::state(c.v), stream);
            }
            op_launch(select, device, stream, {static_cast<uint32_t>(rows * f.cluster), 1, 1},
                      static_cast<uint32_t>(f.threads), sparams, static_cast<uint32_t>(f.cluster));
            if (move != nullptr)
                op_launch(*move, device, stream, {static_cast<uint32_t>(blocks), 1, 1}, 256, mparams);
        }
        return {finish(std::move(os)), finish(std::move(op))};
    }

    void paged_cache_sources(kernel_list& out) {
        kv_cache c;
        c.heads = 5;
        c.dim = 80;
        c.page_size = 8;
        for (const auto type : {cache_type::f32, cache_type::bf16}) {
            c.type = type;
            const std::string tag = type == cache_type::bf16 ? "_bf16" : "_f32", p = kernel_prelude();
            out.emplace_back("pb_cache_append" + tag, p + defines(c, type == cache_type::bf16) + append_source());
            out.emplace_back("pb_evict" + tag, p + defines(c, true) + evict_source());
            out.emplace_back("pb_evict_select" + tag, p + defines(c, true, type == cache_type::bf16 ? select_shape{8, 1024, 48} : select_shape{1, 256, 4}) + evict_source());
            out.emplace_back("pb_evict_select_long" + tag, p + defines(c, true, {8, 1024, 4, false}) + evict_source());
        }
    }

} // namespace porch::detail
