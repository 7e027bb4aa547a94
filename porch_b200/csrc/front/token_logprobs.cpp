// What a row of logits x says of its tokens, in one pass over it, and the
// gradient. With m = max x, s = sum exp(x - m) and w = sum exp(x - m) (x - m):
//   log p(t) = x_t - m - log s,   H = log s - w / s,
// beside the `top` largest logits (equal ones: the lower token). From the
// gradients g of log p(t) and h of H:
//   dx_i = g ([i = t] - p_i) - h p_i (log p_i + H).
//
// Bound: HBM, 4 bytes a logit forward and 8 in the gradient. A thread holds 16
// logits at a time and a running (m, s, w), which is rescaled where their
// maximum is a new one. Sums are fp32: 16 logits in two chains, 32 such rounds one
// after the other, then a thread's blocks of 32 rounds (one for each 2^17 logits of a
// row where rows are many, so at most 128), then threads pairwise; each addition
// rounds, so s and w are within some (60 + V / 2^17) 2^-24 of themselves, and a term
// by 2^-22 more (ex2) and 2^-23 |x - m|. log p and H are so good to about 1e-7
// absolutely, not relative to a log p near 0. One launch: a row that few others keep company is shared
// out over a cluster, whose first CTA joins the parts from the others' shared
// memory. 4093 x 50257: 138 us = 6.0 TB/s; its gradient at 4096 x 65536: 339 us =
// 6.3 TB/s (a call, inputs rotated past the L2 cache). Few rows are bound by latencies:
// 64 x 131072 with the 20 largest 17 to 21 us of the stream (10.6 without), one row of
// 32000 with 5 of them 7 us.
#include "operators.hpp"

#include <algorithm>
#include <sstream>
#include <stdexcept>

namespace porch::detail {

    namespace {

        void expect(bool ok, const char* message) {
            if (!ok) throw std::invalid_argument(message);
        }

        const char* device_source() {
            return R"PB(
typedef long long pb_i64;
#define PB_WARPS (PB_THREADS / 32)
#define PB_LOWEST __int_as_float(0xff7fffff)
#define PB_NAN __int_as_float(0x7fffffff)
#define PB_LOG2E 1.4426950408889634f

static __device__ __forceinline__ float pb_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Finite where x is -inf, so that a weight of 0 times it is 0.
static __device__ __forceinline__ float pb_finite(float x) { return fmaxf(x, -1e30f); }

// Four values of the row from element 4 j - shift on (`shift` of them lie
// before the row, so that the others start on 16 bytes); `none` outside it.
static __device__ __forceinline__ float4 pb_four(const float* row, int at, int n, float none) {
    if (at >= 0 && at + 4 <= n) return __ldcs(reinterpret_cast<const float4*>(row + at));
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = at + e >= 0 && at + e < n ? __ldg(row + at + e) : none;
    return make_float4(v[0], v[1], v[2], v[3]);
}

// What the tokens' numbers say: the token, -1 for a padded row, -2 for anything else.
static __device__ __forceinline__ int pb_token(float t, int V) {
    if (t == -1.0f) return -1;
    return t >= 0.0f && t < (float)V && t == truncf(t) ? (int)t : -2;
}

#ifdef PB_FORWARD
struct pb_sums { float m, s, w; };
static __device__ __forceinline__ void pb_rescale(pb_sums& a, float m) {
    const float d = pb_finite(a.m - m), c = pb_exp2(d * PB_LOG2E);
    a.w = fmaf(a.s, d, a.w) * c;
    a.s *= c;
    a.m = m;
}
static __device__ __forceinline__ pb_sums pb_join(pb_sums a, pb_sums b) {
    const float m = fmaxf(a.m, b.m);
    pb_rescale(a, m);
    pb_rescale(b, m);
    a.s += b.s;
    a.w += b.w;
    return a;
}

static __device__ __forceinline__ pb_u32 pb_rank() {
    pb_u32 r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
static __device__ __forceinline__ void pb_cluster_sync() {
#if PB_CLUSTER > 1
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
#endif
}
// A word of CTA `rank` of the cluster.
static __device__ __forceinline__ pb_u32 pb_peer(const void* p, pb_u32 rank) {
    pb_u32 v, a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((pb_u32)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

#if PB_TOP
// A logit and its token as one number that orders as alternatives do: larger
// logits first (NaN last), of equal ones the lower token. 0 is no entry.
static __device__ __forceinline__ pb_u32 pb_order(float x) {
    const pb_u32 u = __float_as_uint(x + 0.0f); // -0 becomes 0
    return x == x ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 1u;
}
// -inf for NaN and for no entry.
static __device__ __forceinline__ float pb_unorder(pb_u32 k) {
    return k <= 1u ? __int_as_float(0xff800000) : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
static __device__ __forceinline__ pb_u64 pb_key(float x, pb_u32 token) {
    return (pb_u64)pb_order(x) << 32 | (0xffffffffu - token);
}
static __device__ __forceinline__ float pb_logit(pb_u64 key) {
    return (pb_u32)(key >> 32) <= 1u ? PB_NAN : pb_unorder((pb_u32)(key >> 32));
}
// A warp's list: the largest keys so far in falling order, one a lane.
static __device__ __forceinline__ void pb_insert(pb_u64& list, pb_u64 key, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, list > key)); // falling: a run of lanes from 0
    const pb_u64 above = __shfl_up_sync(0xffffffffu, list, 1);
    if (lane >= at) list = lane == at ? key : above;
}
// The 32 largest of two such lists: the larger of entry i and the other's entry
// 31 - i, which rise and then fall, sorted by halving distances.
template <typename T>
static __device__ __forceinline__ T pb_merge(T a, T b, int lane) {
    const T r = __shfl_xor_sync(0xffffffffu, b, 31);
    a = a > r ? a : r;
#pragma unroll
    for (int m = 16; m > 0; m /= 2) {
        const T o = __shfl_xor_sync(0xffffffffu, a, m);
        a = ((lane & m) == 0) == (a > o) ? a : o;
    }
    return a;
}
// Sorts one key a lane, falling.
template <typename T>
static __device__ __forceinline__ T pb_sorted(T a, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int m = size / 2; m > 0; m /= 2) {
            const T o = __shfl_xor_sync(0xffffffffu, a, m);
            const bool keep_larger = ((lane & m) == 0) == ((lane & size) == 0);
            a = keep_larger == (a > o) ? a : o;
        }
    return a;
}
#endif

// A thread's 16 logits of the round at vector `base`; -inf outside the run and the row.
static __device__ __forceinline__ void pb_load(float* v, const float* x, int base, int last, int shift, int V, bool on) {
    const float none = __int_as_float(0xff800000);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int j = base + q * PB_THREADS + threadIdx.x;
        const float4 f = on && j < last ? pb_four(x, 4 * j - shift, V, none) : make_float4(none, none, none, none);
        v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
    }
}

// Cluster: one row, each CTA a run of `run` vectors of it.
extern "C" __global__ void __launch_bounds__(PB_THREADS, 1024 / PB_THREADS) pb_token_logprobs(
    const float* logits, const float* tokens, float* said, float* entropy, float* norm, float* top_said, float* top_tokens,
    int V, pb_i64 stride, int run, int top) { // a vocabulary is below 2^25, and so is every place in it
    __shared__ float sums[PB_WARPS][3];
#if PB_TOP
    __shared__ pb_u64 lists[PB_WARPS][32];
    __shared__ pb_u32 groups[PB_THREADS];
    __shared__ int listed;
#endif
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_u32 row = blockIdx.x / PB_CLUSTER, rank = PB_CLUSTER > 1 ? pb_rank() : 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* x = logits + (pb_i64)row * stride;
    const int shift = (int)(reinterpret_cast<pb_u64>(x) >> 2 & 3);
    const int vectors = (V + shift + 3) >> 2, first = (int)rank * run, last = min(vectors, first + run);
    pb_sums a = {PB_LOWEST, 0.0f, 0.0f};
#if PB_BLOCKS
    pb_sums blocks = a;
    int rounds = 0; // of this block
#endif
#if PB_TOP
    // This lane's largest of a round, that round, and the largest of the others.
    float m1 = __int_as_float(0xff800000), m2 = m1;
    int b1 = first;
#endif
#pragma unroll 1
    for (int base = first; base < last; base += 4 * PB_THREADS) {
        float v[16];
        pb_load(v, x, base, last, shift, V, true);
        float most = v[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) most = fmaxf(most, v[e]);
        if (most > a.m) pb_rescale(a, most);
        float s[2] = {0.0f, 0.0f}, w[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float d = v[e] - a.m, p = pb_exp2(d * PB_LOG2E);
            s[e & 1] += p;
            w[e & 1] = fmaf(p, pb_finite(d), w[e & 1]);
        }
        a.s += s[0] + s[1];
        a.w += w[0] + w[1];
#if PB_BLOCKS
        if (++rounds == 32) { // sums of sums, so that few additions follow each other
            blocks = pb_join(blocks, a);
            a.s = a.w = 0.0f;
            rounds = 0;
        }
#endif
#if PB_TOP
        if (most > m1) { m2 = m1; m1 = most; b1 = base; }
        else m2 = fmaxf(m2, most);
#endif
    }
#if PB_BLOCKS
    a = pb_join(blocks, a);
#endif
#if PB_TOP
    // The alternatives. The largest of a group of logits stands for one of them, so
    // the `top`-th largest of 64 groups' is a floor for all; with the CTA's logits
    // in 64 groups some 24 lie at or above it for 20 alternatives and 44 for 32,
    // whatever their number. The lanes that have some look at them once more (where the largest of
    // a lane's other rounds is below the floor, at one round alone) and list them;
    // NaN is none. The list is then sorted, 32 a warp. Only where it is too long,
    // as of a row of equal logits, or where fewer than `top` of a CTA's groups hold one
    // that is not masked, they are inserted one by one (64 x 131072, 20 alternatives:
    // 64 us with all but 50 masked, 16.5 with all but 2000).
    pb_u64 list = 0;
    int lists_used = 0;
    if (last > first) { // the same for the whole CTA
        groups[threadIdx.x] = pb_order(m1);
        if (threadIdx.x == 0) listed = 0;
        __syncthreads();
        pb_u32 mine[2] = {0, 0};
#pragma unroll
        for (int w = 0; w < PB_WARPS; ++w) mine[w & 1] = max(mine[w & 1], groups[w * 32 + lane]);
        const pb_u32 largest = pb_merge(pb_sorted(mine[0], lane), pb_sorted(mine[1], lane), lane);
        const float low = pb_unorder(__shfl_sync(0xffffffffu, largest, top - 1));
        if (m1 >= low)
            for (int base = m2 >= low ? first : b1; base < last; base += 4 * PB_THREADS) {
                float v[16];
                pb_load(v, x, base, last, shift, V, true);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (v[e] >= low) {
                        const int j = base + (e >> 2) * PB_THREADS + threadIdx.x, at = 4 * j - shift + (e & 3);
                        if (j < last && at >= 0 && at < V) {
                            const int place = atomicAdd(&listed, 1);
                            if (place < PB_THREADS) lists[place / 32][place % 32] = pb_key(v[e], (pb_u32)at);
                        }
                    }
                if (m2 < low) break;
            }
        __syncthreads();
        const int count = listed;
        if (count <= PB_THREADS) {
            lists_used = (count + 31) / 32;
            if (warp < lists_used) list = pb_sorted(32 * warp + lane < count ? lists[warp][lane] : 0, lane);
        } else {
            lists_used = PB_WARPS;
            pb_u64 least = 0; // the list's entry `top` - 1
#pragma unroll 1
            for (int base = first; base < last; base += 4 * PB_THREADS) {
                float v[16];
                pb_load(v, x, base, last, shift, V, m1 >= low);
#pragma unroll 1
                for (int e = 0; e < 16; ++e) {
                    float y = v[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) y = i == e ? v[i] : y;
                    const int j = base + (e >> 2) * PB_THREADS + threadIdx.x, at = 4 * j - shift + (e & 3);
                    const pb_u64 key = y >= low && j < last && at >= 0 && at < V ? pb_key(y, (pb_u32)at) : 0;
                    for (pb_u32 wanting = __ballot_sync(0xffffffffu, key > least); wanting != 0;) {
                        pb_insert(list, __shfl_sync(0xffffffffu, key, __ffs(wanting) - 1), lane);
                        least = __shfl_sync(0xffffffffu, list, top - 1);
                        wanting = (wanting & (wanting - 1)) & __ballot_sync(0xffffffffu, key > least);
                    }
                }
            }
        }
    }
#endif
    asm volatile("griddepcontrol.launch_dependents;");
#pragma unroll
    for (int m = 16; m > 0; m /= 2) {
        const pb_sums o = {__shfl_xor_sync(0xffffffffu, a.m, m), __shfl_xor_sync(0xffffffffu, a.s, m),
                           __shfl_xor_sync(0xffffffffu, a.w, m)};
        a = pb_join(a, o);
    }
    if (lane == 0) { sums[warp][0] = a.m; sums[warp][1] = a.s; sums[warp][2] = a.w; }
#if PB_TOP
    __syncthreads();
    lists[warp][lane] = list;
    // The lists in pairs, pairs of pairs, ...
    for (int m = 1; m < lists_used; m *= 2) {
        __syncthreads();
        if (warp % (2 * m) == 0 && warp + m < lists_used) {
            list = pb_merge(list, lists[warp + m][lane], lane);
            lists[warp][lane] = list;
        }
    }
#endif
    __syncthreads();
    if (warp == 0) {
        a = lane < PB_WARPS ? pb_sums{sums[lane][0], sums[lane][1], sums[lane][2]} : pb_sums{PB_LOWEST, 0.0f, 0.0f};
#pragma unroll
        for (int m = PB_WARPS / 2; m > 0; m /= 2) {
            const pb_sums o = {__shfl_xor_sync(0xffffffffu, a.m, m), __shfl_xor_sync(0xffffffffu, a.s, m),
                               __shfl_xor_sync(0xffffffffu, a.w, m)};
            a = pb_join(a, o);
        }
        __syncwarp();
        if (lane == 0) { sums[0][0] = a.m; sums[0][1] = a.s; sums[0][2] = a.w; }
    }
    pb_cluster_sync();
    if (rank == 0 && warp == 0) {
#if PB_CLUSTER > 1
        if (lane < PB_CLUSTER) a = {__uint_as_float(pb_peer(&sums[0][0], lane)), __uint_as_float(pb_peer(&sums[0][1], lane)),
                                    __uint_as_float(pb_peer(&sums[0][2], lane))};
        else a = {PB_LOWEST, 0.0f, 0.0f};
#pragma unroll
        for (int m = PB_CLUSTER / 2; m > 0; m /= 2) {
            const pb_sums o = {__shfl_xor_sync(0xffffffffu, a.m, m), __shfl_xor_sync(0xffffffffu, a.s, m),
                               __shfl_xor_sync(0xffffffffu, a.w, m)};
            a = pb_join(a, o);
        }
#endif
        a = {__shfl_sync(0xffffffffu, a.m, 0), __shfl_sync(0xffffffffu, a.s, 0), __shfl_sync(0xffffffffu, a.w, 0)};
        const bool good = a.s > 0.0f; // not: nothing but -inf, or a NaN or +inf
        const float total = good ? a.s : PB_NAN, log_total = logf(total);
        if (lane == 0) {
            const int t = pb_token(__ldg(tokens + row), V);
            said[row] = t >= 0 ? (__ldg(x + t) - a.m) - log_total : (t == -1 ? 0.0f : PB_NAN);
            entropy[row] = log_total - a.w / total;
            norm[2 * (pb_i64)row] = a.m;
            norm[2 * (pb_i64)row + 1] = total;
        }
#if PB_TOP
#if PB_CLUSTER > 1
        pb_u64 of[PB_CLUSTER];
        of[0] = list;
#pragma unroll
        for (int c = 1; c < PB_CLUSTER; ++c)
            of[c] = (pb_u64)pb_peer(reinterpret_cast<const pb_u32*>(&lists[0][lane]) + 1, c) << 32 | pb_peer(&lists[0][lane], c);
#pragma unroll
        for (int m = 1; m < PB_CLUSTER; m *= 2)
#pragma unroll
            for (int c = 0; c < PB_CLUSTER; c += 2 * m) of[c] = pb_merge(of[c], of[c + m], lane);
        list = of[0];
#endif
        // Fewer numbers than alternatives: NaN comes last, in order.
        if (__shfl_sync(0xffffffffu, list, top - 1) == 0)
            for (int i = 0; i < V; i += 32) {
                const float y = i + lane < V ? __ldg(x + i + lane) : 0.0f;
                for (pb_u32 nans = __ballot_sync(0xffffffffu, y != y); nans != 0; nans &= nans - 1)
                    pb_insert(list, pb_key(PB_NAN, (pb_u32)(i + __ffs(nans) - 1)), lane);
            }
        if (lane < top) {
            top_said[(pb_i64)row * top + lane] = (pb_logit(list) - a.m) - log_total;
            top_tokens[(pb_i64)row * top + lane] = (float)(0xffffffffu - (pb_u32)list);
        }
#endif
    }
    pb_cluster_sync(); // nobody leaves while its shared memory is read
}
#endif

#ifdef PB_BACKWARD
// Block: PB_LOOPS times 4096 gradients of one row, 16 a thread at once. Where there
// are many, four times: what the row has one of is loaded once for them (4096 x
// 65536: 322 us, 327 with one; 37 x 50257, cold: 14.8, 12.6 with one). Five blocks
// of an SM at once (324 us with four, and with six).
//
// e^d = 2^b e^(d - b log 2) for any b, here d log2 e rounded; what the rounding
// left is so small that e to it is 1 plus it (two terms of log 2 take the
// difference), so p is within a few units of its last place also far below the
// maximum. Below e^-200, which float32 has no number for, every d counts as -200.
// The row's scale, sign and constants are folded into two numbers outside the loop,
// since the instructions show: 322 us, 349 with them taken at each logit.
#define PB_ROUNDS 4
extern "C" __global__ void __launch_bounds__(256, 5) pb_token_logprobs_grad(
    const float* d_said, const float* d_entropy, const float* logits, const float* tokens, const float* norm,
    const float* entropy, float* out, int V, pb_i64 stride, pb_u32 blocks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_u32 row = blockIdx.x / blocks;
    const float* x = logits + (pb_i64)row * stride;
    float* to = out + (pb_i64)row * V;
    const int shift = (int)(reinterpret_cast<pb_u64>(to) >> 2 & 3);
    const bool same = (int)(reinterpret_cast<pb_u64>(x) >> 2 & 3) == shift; // the stores are aligned, the loads where they can be
    const int t = pb_token(__ldg(tokens + row), V);
    const float m = __ldg(norm + 2 * (pb_i64)row), s = __ldg(norm + 2 * (pb_i64)row + 1);
    const float g = t >= 0 ? __ldg(d_said + row) : (t == -1 ? 0.0f : PB_NAN);
#if PB_ENTROPY
    // -p (g + h (d - log s + H)) = -p (c + h d)
    const float h = __ldg(d_entropy + row), c = fmaf(h, __ldg(entropy + row) - logf(s), g), scale = -1.0f / s;
    const bool nothing = t == -1 && h == 0.0f; // a padded row, whatever it holds
#else
    const float scale = -g / s;
    const bool nothing = t == -1;
#endif
    int first = (int)(blockIdx.x % blocks) * (PB_LOOPS * PB_ROUNDS * 256) + threadIdx.x;
#pragma unroll 1
    for (int loop = 0; loop < PB_LOOPS; ++loop, first += PB_ROUNDS * 256) {
        float4 v[PB_ROUNDS];
#pragma unroll
        for (int q = 0; q < PB_ROUNDS; ++q) {
            const int at = 4 * (first + q * 256) - shift;
            if (at >= V || nothing) {
                v[q] = make_float4(m, m, m, m);
            } else if (same) {
                v[q] = pb_four(x, at, V, 0.0f);
            } else {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = at + i >= 0 && at + i < V ? __ldg(x + at + i) : 0.0f;
                v[q] = make_float4(e[0], e[1], e[2], e[3]);
            }
        }
#pragma unroll
        for (int q = 0; q < PB_ROUNDS; ++q) {
            const int at = 4 * (first + q * 256) - shift;
            if (at >= V) break;
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float rel = fmaxf(pb_get(v[q], e) - m, -200.0f), b = rel * PB_LOG2E;
                const float left = fmaf(b, 1.90465432e-09f, fmaf(b, -0.693147182f, rel));
                const float z = pb_exp2(b) * scale;
                const float p = fmaf(z, left, z);
#if PB_ENTROPY
                d[e] = p * fmaf(h, rel, c);
#else
                d[e] = p;
#endif
                if (nothing) d[e] = 0.0f;
            }
            if ((pb_u32)(t - at) < 4u)
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] += at + e == t ? g : 0.0f;
            if (at >= 0 && at + 4 <= V) {
                __stcs(reinterpret_cast<float4*>(to + at), make_float4(d[0], d[1], d[2], d[3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e >= 0 && at + e < V) to[at + e] = d[e];
            }
        }
    }
}
#endif
)PB";
        }

        // How rows are shared out.
        struct shape {
            int cluster = 1, threads = 256;
            bool top = false;
            bool blocks = false; // a thread has more than 32 rounds, whose sums are taken in blocks
        };

        // CTAs of a row: more as long as they all run at once and each thread
        // has its 16 logits; and threads of a CTA, more where an SM has one.
        shape shape_for(int64_t rows, int64_t vocab, bool top, int sms) {
            shape r;
            r.top = top;
            while (r.cluster < 8 && rows * r.cluster * 2 <= int64_t{4} * sms && vocab >= int64_t{r.cluster} * 2 * 4096) r.cluster *= 2;
            while (r.threads < 1024 && rows * r.cluster * r.threads * 2 <= int64_t{1024} * sms &&
                   vocab >= int64_t{r.cluster} * r.threads * 32)
                r.threads *= 2;
            // (4093 x 50257, 13 rounds: 139.4 us a call with blocks, 138.1 without.)
            r.blocks = (vocab + 6) / 4 > int64_t{32} * 4 * r.cluster * r.threads;
            return r;
        }

        std::string forward_source(const shape& f) {
            std::ostringstream os;
            os << kernel_prelude() << "#define PB_FORWARD 1\n#define PB_CLUSTER " << f.cluster << "\n#define PB_THREADS "
               << f.threads << "\n#define PB_TOP " << (f.top ? 1 : 0) << "\n#define PB_BLOCKS " << (f.blocks ? 1 : 0) << "\n"
               << device_source();
            return os.str();
        }

        std::string backward_source(bool entropy, int loops) {
            std::ostringstream os;
            os << kernel_prelude() << "#define PB_BACKWARD 1\n#define PB_THREADS 256\n#define PB_ENTROPY " << (entropy ? 1 : 0)
               << "\n#define PB_LOOPS " << loops << "\n" << device_source();
            return os.str();
        }

        const char kForward[] = "pb_token_logprobs";
        const char kBackward[] = "pb_token_logprobs_grad";

        op_kernel& forward_kernel(const shape& f) {
            const op_key key{reinterpret_cast<int64_t>(kForward), f.cluster, f.threads, f.top, f.blocks};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = kForward;
                k.source = forward_source(f);
            });
        }

        op_kernel& backward_kernel(bool entropy, int loops) {
            const op_key key{reinterpret_cast<int64_t>(kBackward), entropy, loops};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = kBackward;
                k.source = backward_source(entropy, loops);
            });
        }

        // [rows, vocabulary] of logits, and a token of each row.
        void check_logits(const tensor& logits, const tensor& tokens) {
            const auto s = logits.shape();
            expect(s.size() == 2, "token_logprobs: logits must be [rows, vocabulary]");
            expect(s[1] >= 1 && s[1] <= (index_t{1} << 24), "token_logprobs: a vocabulary of 1 to 2^24 tokens (float32 counts them exactly)");
            expect(has_shape(tokens, {s[0]}), "token_logprobs: tokens must be [rows]");
        }

    } // namespace

    std::vector<tensor> token_logprobs(const tensor& logits, const tensor& tokens, int64_t top) {
        check_logits(logits, tokens);
        const auto s = shape_of(logits);
        expect(top >= 0 && top <= 32 && top <= s[1], "token_logprobs: top must be 0 to 32, and at most the vocabulary");
        const int device = device_of(logits, "token_logprobs");
        expect(device_of(tokens, "token_logprobs") == device, "token_logprobs: operands must live on one device");
        auto stream = current_stream(device);
        op_operand x = operand(logits, stream, true), t = operand(tokens, stream, false);
        const int64_t rows = s[0], vocab = s[1];
        int V = static_cast<int>(vocab);
        op_result said = new_result({rows}, device, stream), entropy = new_result({rows}, device, stream);
        op_result norm = new_result({rows, 2}, device, stream);
        op_result top_said, top_tokens;
        if (top != 0) {
            top_said = new_result({rows, top}, device, stream);
            top_tokens = new_result({rows, top}, device, stream);
        }
        if (rows != 0) {
            const shape f = shape_for(rows, vocab, top != 0, sm_count(device));
            op_kernel& kernel = forward_kernel(f);
            expect(rows <= 0x7fffffff / f.cluster, "token_logprobs: too many rows");
            // Vectors of a CTA: with up to three values before the row's first.
            int run = static_cast<int>(((vocab + 6) / 4 + f.cluster - 1) / f.cluster), most = static_cast<int>(top);
            int64_t stride = rows > 1 ? x.strides[0] : vocab;
            void* params[] = {&x.ptr,        &t.ptr,          &said.ptr, &entropy.ptr, &norm.ptr, &top_said.ptr,
                              &top_tokens.ptr, &V,            &stride,   &run,         &most};
            op_launch(kernel, device, stream, {static_cast<uint32_t>(rows * f.cluster), 1, 1},
                      static_cast<uint32_t>(f.threads), params, static_cast<uint32_t>(f.cluster));
        }
        std::vector<tensor> out;
        out.push_back(finish(std::move(said)));
        out.push_back(finish(std::move(entropy)));
        out.push_back(finish(std::move(norm)));
        if (top != 0) {
            out.push_back(finish(std::move(top_said)));
            out.push_back(finish(std::move(top_tokens)));
        }
        return out;
    }

    tensor token_logprobs_backward(const tensor& d_said, const tensor& logits, const tensor& tokens, const tensor& norm,
                                   const tensor* d_entropy, const tensor* entropy) {
        check_logits(logits, tokens);
        const auto s = shape_of(logits);
        expect(has_shape(d_said, {s[0]}), "token_logprobs_backward: d_logprobs must be [rows]");
        expect(has_shape(norm, {s[0], 2}), "token_logprobs_backward: norm must be [rows, 2], as token_logprobs gave it");
        expect((d_entropy != nullptr) == (entropy != nullptr), "token_logprobs_backward: d_entropy needs entropy, and entropy d_entropy");
        expect(d_entropy == nullptr || (has_shape(*d_entropy, {s[0]}) && has_shape(*entropy, {s[0]})),
               "token_logprobs_backward: d_entropy and entropy must be [rows]");
        const int device = device_of(logits, "token_logprobs_backward");
        auto stream = current_stream(device);
        op_operand x = operand(logits, stream, true), t = operand(tokens, stream, false), g = operand(d_said, stream, false),
                   n = operand(norm, stream, false), h, e;
        if (d_entropy != nullptr) {
            h = operand(*d_entropy, stream, false);
            e = operand(*entropy, stream, false);
        }
        op_result out = new_result(s, device, stream);
        const int64_t rows = s[0], vocab = s[1];
        int V = static_cast<int>(vocab);
        if (rows != 0) {
            const int64_t vectors = (vocab + 6) / 4; // with up to three values before the row's first
            const int loops = rows * (vectors / 4096) >= int64_t{16} * sm_count(device) ? 4 : 1;
            op_kernel& kernel = backward_kernel(d_entropy != nullptr, loops);
            uint32_t per_row = static_cast<uint32_t>((vectors + 1024 * loops - 1) / (1024 * loops));
            expect(rows <= 0x7fffffff / static_cast<int64_t>(per_row), "token_logprobs_backward: too many rows");
            int64_t stride = rows > 1 ? x.strides[0] : vocab;
            void* params[] = {&g.ptr, &h.ptr, &x.ptr, &t.ptr, &n.ptr, &e.ptr, &out.ptr, &V, &stride, &per_row};
            op_launch(kernel, device, stream, {static_cast<uint32_t>(rows * per_row), 1, 1}, 256, params);
        }
        return finish(std::move(out));
    }

    void token_logprobs_sources(kernel_list& out) {
        for (const shape& f : {shape{1, 256, false}, shape{1, 256, true, true}, shape{8, 1024, true}, shape{4, 512, false}})
            out.emplace_back("pb_token_logprobs_" + std::to_string(f.cluster) + "x" + std::to_string(f.threads) + (f.top ? "_top" : ""),
                             forward_source(f));
        out.emplace_back("pb_token_logprobs_grad", backward_source(false, 1));
        out.emplace_back("pb_token_logprobs_grad_entropy", backward_source(true, 4));
    }

} // namespace porch::detail
