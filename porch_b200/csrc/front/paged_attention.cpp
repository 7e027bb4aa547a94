// Attention of one new token per sequence over a paged cache:
//   o = softmax(scale q K^T) V
// over the slots in use, query heads sharing key heads in groups, and its
// scored form, which adds each slot's attention weight, summed over the query
// heads of its key head, to running scores (what eviction ranks slots by).
// A sequence without slots gives zeros.
//
// Bound: HBM, which has to deliver every key and value in use once (2 x slots
// x kv_heads x head_dim x 2 or 4 bytes). 48 sequences up to 8191 slots, 32
// query heads over 8 of 128 bfloat16 channels: 784 MB in 126 us = 6.20 TB/s;
// one sequence of 262147 slots: 1074 MB in 165 us = 6.5 TB/s, what a copy
// reaches. Few or short rows are bound by the launch and the first loads'
// latency instead (about 6 us, 3 of the stream where calls follow each other).
//
// pb_paged_attention, 160 threads: a producer warp loads tiles of 64 slots, K
// then V, through a ring of TMA boxes (a page, or 64 rows of a larger one; 128
// bytes wide, swizzled, zeros past the head size), and four computing warps
// keep an online softmax over them: S^T = K Q^T for 16 slots each, a maximum
// over the tile, weights to shared memory, O^T += V^T P^T for a quarter of the
// channels each. The transposed products put slots and channels on the tensor
// core's 16 rows and query heads on its 8 columns, so 1 to 8 heads cost the
// same. One query per sequence leaves nothing for the 128-row tiles of
// tcgen05; with mma.sync the tensor pipe is 31 % busy at full bandwidth.
//
// Accuracy: float32. Queries and weights are split into three bfloat16 terms
// (24 bits) against a bfloat16 cache, whose products are then exact; a float32
// cache is split into two tf32 terms like the queries (each off by up to 2^-21,
// and of four products the smallest is left out: 2^-19.6 of a product at most).
// The tensor core's accumulator cuts low bits at every addition, so a tile's
// products start from zero and are added to the running sums in fp32, rounded to
// nearest.
//
// Work is shared out in even runs of tiles over all rows, one wave of CTAs
// (more waves, which would even out CTAs of different speed, took 1 to 5 %
// longer), and rows that span CTAs are joined from their parts in order, so
// results depend on the lengths and the number of SMs alone. Joining in the
// CTA that finishes a row's last part instead of a second launch took 2 to 13
// us longer: its fences and loads come at the very end.
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <sstream>
#include <stdexcept>

namespace porch::detail {

    namespace {

        void expect(bool ok, const std::string& message) {
            if (!ok) throw std::invalid_argument(message);
        }

        // The whole layout of a kernel follows from these.
        struct form {
            int heads = 1, dim = 0, page = 0;
            bool bf16 = false, scored = false;
            int stall = 0; // the test hook's mode
            int join_threads = 128;
            int tiles8 = 1; // groups of 8 query heads that a row holds (1 or 2)
            int width() const { return bf16 ? 2 : 4; }
            int planes() const { return (dim * width() + 127) / 128; }
            int unit() const { return planes() * 8192; }                       // 64 slots of K or of V
            int steps() const { return ((dim * width() + 31) / 32 + 1) & ~1; } // 32-byte k-steps, an even number
            int terms() const { return bf16 ? 3 : 2; }
            int q_row() const { return steps() * 32 + 16; }
            int p_row() const { return 64 * width() + 16; }
            int small() const { // everything but the ring
                return terms() * tiles8 * 8 * (q_row() + p_row()) + 2 * 4 * tiles8 * 8 * 4;
            }
            int per_sm() const { return choose().first; }
            int ring() const { return choose().second; }
            int chunks(int group) const { return (group + 8 * tiles8 - 1) / (8 * tiles8); } // rows of a key head
            int smem() const { return 1024 + ring() * unit() + small(); }
            // What a CTA takes of an SM's 228 KB: that, the kernel's static
            // arrays (the ring's barriers and a flag, which the kernel checks
            // against kStatic) with the rounding of the sum, and the KB that
            // the system keeps for each CTA.
            static constexpr int kStatic = 256;
            int shared() const { return smem() + kStatic + 1024; }

          private:
            // CTAs of an SM and units of a CTA's ring: as many CTAs as leave
            // room for three units each, so that one is on its way while two
            // are read. CTAs hide each other's barriers (48 sequences up to
            // 8191 slots, 128 bfloat16 channels: 134 us with two CTAs of six
            // units, 124 with three of three).
            std::pair<int, int> choose() const {
                for (int n = 4; n > 1; --n) {
                    const int r = ((228 * 1024) / n - 2048 - kStatic - small()) / unit();
                    if (r >= 3) return {n, std::min(r, 6)};
                }
                return {1, std::min((227 * 1024 - 1024 - kStatic - small()) / unit(), 6)};
            }
        };

        const char* device_source() {
            return R"PB(
typedef long long pb_i64;
#define PB_WAIT_CYCLES 4000000000ll
#define PB_HT (8 * PB_NT)                // query heads of a row, padded
#define PB_PLANES ((PB_D * PB_ESZ + 127) / 128)
#define PB_UNIT (PB_PLANES * 8192)       // 64 slots, one 128-byte plane after the other
#define PB_CE (128 / PB_ESZ)             // values of a plane's row
#define PB_BOX (PB_PS < 64 ? PB_PS : 64) // slots of one tile load
#define PB_STEPS ((((PB_D * PB_ESZ + 31) / 32) + 1) & ~1)
#define PB_QROW (PB_STEPS * 32 + 16)
#define PB_PROW (64 * PB_ESZ + 16)
#define PB_MT ((PB_D + 15) / 16)         // 16-channel tiles of the result
#define PB_MTW ((PB_MT + 3) / 4)         // of one warp
#if PB_ESZ == 2
#define PB_TERMS 3
#else
#define PB_TERMS 2
#endif

struct __align__(64) pb_tmap { unsigned long long opaque[16]; };

static __device__ __forceinline__ pb_u32 pb_smem(const void* p) { return (pb_u32)__cvta_generic_to_shared(p); }
static __device__ __forceinline__ void pb_mbar_init(pb_u32 bar, pb_u32 count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
static __device__ __forceinline__ void pb_mbar_arrive(pb_u32 bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
static __device__ __forceinline__ void pb_mbar_expect_tx(pb_u32 bar, pb_u32 bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
static __device__ __forceinline__ pb_u32 pb_mbar_try(pb_u32 bar, pb_u32 parity) {
    pb_u32 ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Records where a wait gave up; the first one stays.
static __device__ __forceinline__ void pb_gave_up(int* err, int site) {
    if (atomicCAS(err, 0, 0x7d00 + site) == 0) {
        err[1] = site;
        err[2] = (int)blockIdx.x;
    }
}
// Bounded wait: false when the budget ran out or another role gave up.
static __device__ __forceinline__ bool pb_wait(pb_u32 bar, pb_u32 parity, volatile int* abort_flag, int* err, int site) {
    if (pb_mbar_try(bar, parity)) return true;
    const long long start = clock64();
    for (;;) {
        if (pb_mbar_try(bar, parity)) return true;
        if (*abort_flag) return false;
        if (clock64() - start > PB_WAIT_CYCLES) {
            *abort_flag = 1;
            pb_gave_up(err, site);
            return false;
        }
    }
}
static __device__ __forceinline__ void pb_tma_load(pb_u32 dst, const pb_tmap* map, pb_u32 bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 :: "r"(dst), "l"((unsigned long long)map), "r"(bar), "r"(x), "r"(y) : "memory");
}
// Named barrier 1 over the 128 computing threads, with an OR of a predicate:
// a wait that ran out anywhere makes all of them leave at the same place.
static __device__ __forceinline__ bool pb_bar_any(bool v) {
    pb_u32 r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, 1, 128, q;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(r) : "r"((pb_u32)v) : "memory");
    return r != 0;
}
static __device__ __forceinline__ float pb_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// What a maximum over logits begins with: the lowest finite value, so that
// logits of -inf (below float32's range) weigh exp2(-inf) = 0 also where a tile
// or a part holds no other; from -inf they would be the NaN of -inf - -inf.
#define PB_LOWEST __int_as_float(0xff7fffff)

static __device__ __forceinline__ void pb_ldm4(pb_u32* r, pb_u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
static __device__ __forceinline__ void pb_ldm4t(pb_u32* r, pb_u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
#if PB_ESZ == 2
static __device__ __forceinline__ void pb_mma(float* c, const pb_u32* a, const pb_u32* b) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// The upper 16 bits of x rounded to nearest even bfloat16.
static __device__ __forceinline__ unsigned short pb_bf16(float x) {
    unsigned short r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(x));
    return r;
}
static __device__ __forceinline__ float pb_value(unsigned short x) { return __uint_as_float((pb_u32)x << 16); }
// x = t0 + t1 + t2, bfloat16 each: 24 bits, so exactly (until t2 underflows).
static __device__ __forceinline__ void pb_split_store(pb_u32 at, pb_u32 step, float x) {
#pragma unroll
    for (int t = 0; t < 3; ++t) {
        const unsigned short h = pb_bf16(x);
        x -= pb_value(h);
        asm volatile("st.shared.u16 [%0], %1;" :: "r"(at + t * step), "h"(h) : "memory");
    }
}
#else
static __device__ __forceinline__ void pb_mma(float* c, const pb_u32* a, const pb_u32* b) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// x = hi + lo: hi is x rounded to tf32 (10 mantissa bits, half up) by integer
// arithmetic, which runs at the full rate that conversions do not have (16 x
// 2049 slots of 64 channels: 37.6 us with cvt.rna, 34.2 so); x - hi
// is exact, and the tensor core reads its upper 10 bits: an error of at most
// 2^-21 |x|, of either sign. A NaN stays one in lo.
static __device__ __forceinline__ void pb_tf32_split(float x, float& hi, float& lo) {
    hi = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
    lo = x - hi;
}
static __device__ __forceinline__ void pb_split_store(pb_u32 at, pb_u32 step, float x) {
    float hi, lo;
    pb_tf32_split(x, hi, lo);
    asm volatile("st.shared.f32 [%0], %1;" :: "r"(at), "f"(hi) : "memory");
    asm volatile("st.shared.f32 [%0], %1;" :: "r"(at + step), "f"(lo) : "memory");
}
// hi and lo of four fragment values.
static __device__ __forceinline__ void pb_split_frag(const pb_u32* a, pb_u32* hi, pb_u32* lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float h, l;
        pb_tf32_split(__uint_as_float(a[i]), h, l);
        hi[i] = __float_as_uint(h);
        lo[i] = __float_as_uint(l);
    }
}
#endif

// Where a row's tiles come from. Rows are (sequence, key head, chunk of query
// heads), tiles 64 slots of a row; a CTA works through a run of tiles.
struct pb_at { int row, tile; int s, h, chunk, length, tiles; };
static __device__ __forceinline__ void pb_enter(pb_at& a, const int* lengths, int chunks) {
    a.chunk = a.row % chunks;
    a.h = (a.row / chunks) % PB_H;
    a.s = a.row / chunks / PB_H;
    a.length = lengths[a.s];
    a.tiles = (a.length + 63) >> 6;
}
// The next tile; skips sequences without slots. True when it is another row's.
static __device__ __forceinline__ bool pb_next(pb_at& a, const int* lengths, int chunks) {
    if (++a.tile < a.tiles) return false;
    a.tile = 0;
    do {
        ++a.row;
        pb_enter(a, lengths, chunks);
    } while (a.tiles == 0);
    return true;
}

// The page that this lane's part of the tile lies in (0 past its slots).
static __device__ __forceinline__ int pb_page(const pb_at& a, const int* tables, int width, int lane) {
    const int first = a.tile * 64 + lane * PB_BOX;
    return lane * PB_BOX < 64 && first < a.length ? tables[(pb_i64)a.s * width + first / PB_PS] : 0;
}

// A row's queries, PB_Q_EACH values of each of 128 threads, every load before
// the first use; zero past its heads and the head size.
#define PB_Q_HEAD (PB_STEPS * 32 / PB_ESZ)
#define PB_Q_EACH ((PB_HT * PB_Q_HEAD + 127) / 128)
struct pb_queries { float x[PB_Q_EACH]; };
static __device__ __forceinline__ void pb_load_queries(pb_queries& r, const float* q, const pb_at& a, pb_i64 q_seq,
                                                       pb_i64 q_head, int group) {
    const int heads = min(PB_HT, group - a.chunk * PB_HT), first = a.h * group + a.chunk * PB_HT;
#pragma unroll
    for (int j = 0; j < PB_Q_EACH; ++j) {
        const int e = threadIdx.x + 128 * j, head = e / PB_Q_HEAD, d = e % PB_Q_HEAD;
        r.x[j] = head < heads && d < PB_D ? __ldg(q + a.s * q_seq + (first + head) * q_head + d) : 0.0f;
    }
}

extern "C" __global__ void __launch_bounds__(160, PB_PER_SM) pb_paged_attention(
    const __grid_constant__ pb_tmap map_k, const __grid_constant__ pb_tmap map_v, const float* q, const int* lengths,
    const int* tables, const int4* work, float* out, float* partial, float2* partial_ml, float* logits, float2* norms,
    int width, int group, int chunks, pb_i64 q_seq, pb_i64 q_head, int longest, float scale2, int* err) {
    extern __shared__ char raw[];
    __shared__ pb_u64 bars[2 * PB_RING];
    __shared__ int abort_flag;
    static_assert(sizeof(bars) + sizeof(abort_flag) + 128 <= PB_STATIC, "shared memory that the launch does not count");
    const pb_u32 ring = (pb_smem(raw) + 1023u) & ~1023u;
    const pb_u32 qs = ring + PB_RING * PB_UNIT;
    const pb_u32 ps = qs + PB_TERMS * PB_HT * PB_QROW;
    float* wmax = reinterpret_cast<float*>(raw + (ps + PB_TERMS * PB_HT * PB_PROW - pb_smem(raw)));
    float* wsum = wmax + 4 * PB_HT;
    const pb_u32 full = pb_smem(bars), empty = full + 8 * PB_RING;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PB_RING; ++i) {
            pb_mbar_init(full + 8 * i, 1);
            pb_mbar_init(empty + 8 * i, 4);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // The plan, lengths and tables were in place before the launch (their
    // upload was waited for on the host), so they are read while the previous
    // kernel still runs; everything else waits for it.
    const int4 mine = work[blockIdx.x];
    pb_at at;
    at.row = mine.x;
    at.tile = mine.y;
    pb_enter(at, lengths, chunks);

    if (warp == 4) {
        // ---- producer: K then V of each tile into the ring
        int slot = 0, unit = 0;
        pb_u32 parity = 1; // the first round finds every unit free
        bool bad = false;
        int page = pb_page(at, tables, width, lane);
        asm volatile("griddepcontrol.wait;" ::: "memory");
#if PB_TEST_STALL == 1
        if (blockIdx.x == 0) return; // its tiles never arrive
#endif
        for (int i = 0; i < mine.z && !bad; ++i) {
            const int base = at.tile * 64, boxes = (min(64, at.length - base) + PB_BOX - 1) / PB_BOX;
            const int y = (page * PB_H + at.h) * PB_PS + (base + lane * PB_BOX) % PB_PS;
            if (i + 1 < mine.z) { // the next tile's pages are looked up while this one's loads are issued
                pb_next(at, lengths, chunks);
                page = pb_page(at, tables, width, lane);
            }
#pragma unroll 1
            for (int which = 0; which < 2 && !bad; ++which) {
                bad = !pb_wait(empty + 8 * slot, parity, &abort_flag, err, 1 + which);
                bad = __any_sync(0xffffffffu, bad);
                if (bad) break;
                if (lane == 0) pb_mbar_expect_tx(full + 8 * slot, boxes * PB_BOX * 128 * PB_PLANES);
                __syncwarp();
                if (lane < boxes) {
                    const pb_u32 dst = ring + slot * PB_UNIT + lane * PB_BOX * 128;
#pragma unroll
                    for (int c = 0; c < PB_PLANES; ++c)
                        pb_tma_load(dst + c * 8192, which ? &map_v : &map_k, full + 8 * slot, c * PB_CE, y);
                }
                ++unit;
                if (++slot == PB_RING) { slot = 0; parity ^= 1u; }
            }
        }
        // Nothing may land after this CTA is gone: wait (bounded) for what is
        // still in flight. Always, since the computing warps may give up after
        // the last load was issued; while they do not, they wait for the same.
        if (lane == 0) {
            for (int u = unit > PB_RING ? unit - PB_RING : 0; u < unit; ++u) {
                const long long start = clock64();
                while (!pb_mbar_try(full + 8 * (u % PB_RING), (u / PB_RING) & 1) && clock64() - start <= PB_WAIT_CYCLES) {
                }
            }
        }
        return;
    }

    // ---- four computing warps
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (mine.z == 0) { // a row without slots
        const int heads = min(PB_HT, group - at.chunk * PB_HT);
        const pb_i64 to = (pb_i64)at.s * PB_H * group + at.h * group + at.chunk * PB_HT;
        for (int e = threadIdx.x; e < heads * PB_D; e += 128) out[to * PB_D + e] = 0.0f;
        return;
    }
    const int g = lane >> 2, t = lane & 3;
    int slot = 0;
    pb_u32 parity = 0;
    bool bad = false, fresh = true;
    int segment = 0; // how many rows this CTA has begun
    float m[PB_NT][2], l[PB_NT][2], o[PB_MTW][PB_NT][4];
    bool begun_at_zero = true;
#if PB_ESZ == 4
    // Where this thread's four values of V^T lie in each of its channel tiles
    // (slots 2 t and 2 t + 1 of a group of 8, channels g and g + 8).
    pb_u32 v_at[PB_MTW][4];
#pragma unroll
    for (int a = 0; a < PB_MTW; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 2 * t + (e >> 1), ch = (warp + 4 * a) * 16 + g + (e & 1) * 8;
            v_at[a][e] = (ch >> 5) * 8192 + r * 128 + ((((ch & 31) >> 2) ^ r) << 4) + (ch & 3) * 4;
        }
#endif
    // The next tile is looked up, and the next row's queries are loaded, a tile
    // ahead, so that neither is waited for (queries only where they take few
    // registers).
    pb_at next = at;
    bool next_fresh = false;
    pb_queries ahead;
    pb_load_queries(ahead, q, at, q_seq, q_head, group);
    for (int i = 0; i < mine.z; ++i) {
        if (i) {
            at = next;
            fresh = next_fresh;
        }
        if (i + 1 < mine.z) next_fresh = pb_next(next, lengths, chunks);
        const int hg = min(PB_HT, group - at.chunk * PB_HT);             // query heads of this row
        const int head0 = at.h * group + at.chunk * PB_HT;                // the first
        if (fresh) {
            begun_at_zero = at.tile == 0;
            // The row's queries, split into terms; zero past the head size.
            if (PB_Q_EACH > 8 && i) pb_load_queries(ahead, q, at, q_seq, q_head, group);
#pragma unroll
            for (int j = 0; j < PB_Q_EACH; ++j) {
                const int e = threadIdx.x + 128 * j, head = e / PB_Q_HEAD, d = e % PB_Q_HEAD;
                if (e < PB_HT * PB_Q_HEAD) pb_split_store(qs + head * PB_QROW + d * PB_ESZ, PB_HT * PB_QROW, ahead.x[j]);
            }
#pragma unroll
            for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) { m[n][e] = PB_LOWEST; l[n][e] = 0.0f; }
#pragma unroll
            for (int a = 0; a < PB_MTW; ++a)
#pragma unroll
                for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[a][n][e] = 0.0f;
            if (pb_bar_any(bad)) { bad = true; break; }
        }
        if (PB_Q_EACH <= 8 && i + 1 < mine.z && next_fresh) pb_load_queries(ahead, q, next, q_seq, q_head, group);
        const int base = at.tile * 64, valid = min(64, at.length - base);

        // ---- S^T = K Q^T: this warp's 16 slots x all heads
#if PB_TEST_STALL == 2
        if (blockIdx.x == 0) { // gives up at once, its first loads on their way
            pb_gave_up(err, 5);
            bad = true;
        } else
#endif
        bad |= !pb_wait(full + 8 * slot, parity, &abort_flag, err, 3);
        // The first term's sum, the large one, runs in two chains that are
        // added in fp32: half the additions that cut bits in a row.
        float c[PB_TERMS + 1][PB_NT][4];
#pragma unroll
        for (int x = 0; x < PB_TERMS + 1; ++x)
#pragma unroll
            for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[x][n][e] = 0.0f;
        {
            const int r = 16 * warp + (lane & 15);
            const pb_u32 krow = ring + slot * PB_UNIT + r * 128;
            const pb_u32 qrow = qs + (lane & 7) * PB_QROW + (lane >> 3) * 16;
#pragma unroll
            for (int k2 = 0; k2 < PB_STEPS / 2; ++k2) {
                pb_u32 a[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int chunk = (2 * k2 + k) * 2; // 16-byte chunk of the row; its plane and place
                    pb_ldm4(a[k], krow + (chunk >> 3) * 8192 + ((((chunk & 7) + (lane >> 4)) ^ (r & 7)) << 4));
                }
#if PB_ESZ == 2
#pragma unroll
                for (int x = 0; x < PB_TERMS; ++x)
#pragma unroll
                    for (int n = 0; n < PB_NT; ++n) {
                        pb_u32 b[4];
                        pb_ldm4(b, qrow + (x * PB_HT + n * 8) * PB_QROW + k2 * 64);
                        pb_mma(c[x][n], a[0], b);
                        pb_mma(c[x == 0 ? PB_TERMS : x][n], a[1], b + 2);
                    }
#else
                pb_u32 hi[2][4], lo[2][4];
                pb_split_frag(a[0], hi[0], lo[0]);
                pb_split_frag(a[1], hi[1], lo[1]);
#pragma unroll
                for (int n = 0; n < PB_NT; ++n) {
                    pb_u32 b[4], b2[4];
                    pb_ldm4(b, qrow + (n * 8) * PB_QROW + k2 * 64);
                    pb_ldm4(b2, qrow + (PB_HT + n * 8) * PB_QROW + k2 * 64);
                    pb_mma(c[0][n], hi[0], b);
                    pb_mma(c[1][n], hi[0], b2);
                    pb_mma(c[PB_TERMS][n], hi[1], b + 2);
                    pb_mma(c[1][n], lo[0], b);
                    pb_mma(c[1][n], hi[1], b2 + 2);
                    pb_mma(c[1][n], lo[1], b + 2);
                }
#endif
            }
        }
        __syncwarp();
        // Not after a wait that gave up: the unit's load may still be on its
        // way, and the producer would issue another one into it.
        if (lane == 0 && !bad) pb_mbar_arrive(empty + 8 * slot);
        if (++slot == PB_RING) { slot = 0; parity ^= 1u; }

        // Logits in units of log2, -inf past the sequence's end. Thread: slots
        // 16 warp + g and + 8, heads 8 n + 2 t and + 1.
        float s[PB_NT][4], top[PB_NT][2];
#pragma unroll
        for (int n = 0; n < PB_NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at_slot = 16 * warp + g + (e >> 1) * 8;
#if PB_TERMS == 3
                const float x = (c[2][n][e] + c[1][n][e] + (c[0][n][e] + c[3][n][e])) * scale2;
#else
                const float x = (c[1][n][e] + (c[0][n][e] + c[2][n][e])) * scale2;
#endif
                s[n][e] = at_slot < valid ? x : __int_as_float(0xff800000);
#if PB_SCORED
                const int head = 8 * n + 2 * t + (e & 1);
                if (at_slot < valid && head < hg)
                    logits[((pb_i64)at.s * PB_H * group + head0 + head) * longest + base + at_slot] = x;
#endif
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(s[n][e], s[n][e + 2]);
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                top[n][e] = x;
            }
            if (g == 0) *reinterpret_cast<float2*>(wmax + warp * PB_HT + 8 * n + 2 * t) = make_float2(top[n][0], top[n][1]);
        }
        if (pb_bar_any(bad)) { bad = true; break; }

        // ---- weights relative to the running maximum, split into terms
        float corr[PB_NT][2];
#pragma unroll
        for (int n = 0; n < PB_NT; ++n) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float2 x = *reinterpret_cast<const float2*>(wmax + w * PB_HT + 8 * n + 2 * t);
                top[n][0] = fmaxf(top[n][0], x.x);
                top[n][1] = fmaxf(top[n][1], x.y);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float now = fmaxf(m[n][e], top[n][e]);
                corr[n][e] = pb_exp2(m[n][e] - now);
                m[n][e] = now;
                l[n][e] *= corr[n][e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = pb_exp2(s[n][e] - m[n][e & 1]);
                l[n][e & 1] += p;
                const int at_slot = 16 * warp + g + (e >> 1) * 8, head = 8 * n + 2 * t + (e & 1);
#if PB_ESZ == 2
                const int place = at_slot;
#else
                const int place = (at_slot & ~7) + ((at_slot & 7) >> 1) + (at_slot & 1) * 4; // as V's fragments count slots
#endif
                pb_split_store(ps + head * PB_PROW + place * PB_ESZ, PB_HT * PB_PROW, p);
            }
        }
        bad |= !pb_wait(full + 8 * slot, parity, &abort_flag, err, 4);
        if (pb_bar_any(bad)) { bad = true; break; }

        // ---- O^T += V^T P^T: this warp's channels x all heads. The tile's sum
        // starts from zero in the tensor core, whose additions cut low bits,
        // and is added to the running one in fp32, rounded to nearest.
        {
            const pb_u32 vunit = ring + slot * PB_UNIT;
            const pb_u32 prow = ps + (lane & 7) * PB_PROW + (lane >> 3) * 16;
            float d[PB_MTW][PB_NT][2][4];
#pragma unroll
            for (int a = 0; a < PB_MTW; ++a)
#pragma unroll
                for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[a][n][0][e] = d[a][n][1][e] = 0.0f;
#pragma unroll
            for (int k2 = 0; k2 < 2 * PB_ESZ / 2; ++k2) { // two k-steps at a time
                pb_u32 b[PB_TERMS][PB_NT][4];
#pragma unroll
                for (int x = 0; x < PB_TERMS; ++x)
#pragma unroll
                    for (int n = 0; n < PB_NT; ++n) pb_ldm4(b[x][n], prow + (x * PB_HT + n * 8) * PB_PROW + k2 * 64);
#pragma unroll
                for (int a = 0; a < PB_MTW; ++a) {
                    const int mt = warp + 4 * a;
                    if (mt < PB_MT) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            pb_u32 v[4];
#if PB_ESZ == 2
                            const int first = (2 * k2 + k) * 16;
                            const int r = first + (lane >> 4) * 8 + (lane & 7);
                            const int chunk = mt * 2 + ((lane >> 3) & 1);
                            pb_ldm4t(v, vunit + (chunk >> 3) * 8192 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
                            if (valid < 64) { // what lies past the end may be anything
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int left = valid - (first + 2 * t + (e >> 1) * 8);
                                    v[e] = left >= 2 ? v[e] : (left == 1 ? v[e] & 0xffffu : 0u);
                                }
                            }
#pragma unroll
                            for (int n = 0; n < PB_NT; ++n) {
                                pb_mma(d[a][n][0], v, b[0][n] + 2 * k);
                                pb_mma(d[a][n][1], v, b[2][n] + 2 * k);
                                pb_mma(d[a][n][1], v, b[1][n] + 2 * k);
                            }
#else
                            // Slots 2 t and 2 t + 1 stand for columns t and t + 4:
                            // their rows' swizzles put the loads on distinct banks.
                            const int first = (2 * k2 + k) * 8 + 2 * t;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                asm volatile("ld.shared.u32 %0, [%1];"
                                             : "=r"(v[e]) : "r"(vunit + v_at[a][e] + (2 * k2 + k) * 1024) : "memory");
                            if (valid < 64) { // what lies past the end may be anything
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (first + (e >> 1) >= valid) v[e] = 0u;
                            }
                            pb_u32 hi[4], lo[4];
                            pb_split_frag(v, hi, lo);
#pragma unroll
                            for (int n = 0; n < PB_NT; ++n) {
                                pb_mma(d[a][n][0], hi, b[0][n] + 2 * k);
                                pb_mma(d[a][n][1], hi, b[1][n] + 2 * k);
                                pb_mma(d[a][n][1], lo, b[0][n] + 2 * k);
                            }
#endif
                        }
                    }
                }
            }
#pragma unroll
            for (int a = 0; a < PB_MTW; ++a)
#pragma unroll
                for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[a][n][e] = fmaf(o[a][n][e], corr[n][e & 1], d[a][n][1][e] + d[a][n][0][e]);
        }
        __syncwarp();
        if (lane == 0) pb_mbar_arrive(empty + 8 * slot);
        if (++slot == PB_RING) { slot = 0; parity ^= 1u; }

        // Only here: joining blocks that come in earlier, or an attention that
        // comes in beside them, take the room of CTAs that are still to run
        // (48 sequences up to 8191 slots: 128 us so, 168 with the launch at
        // every kernel's start).
        if (i + 1 == mine.z) asm volatile("griddepcontrol.launch_dependents;");
        // ---- the row ends, or this CTA's part of it
        const bool row_ends = at.tile + 1 == at.tiles;
        if (row_ends || i + 1 == mine.z) {
#pragma unroll
            for (int n = 0; n < PB_NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = l[n][e];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    l[n][e] = x;
                }
                if (g == 0) *reinterpret_cast<float2*>(wsum + warp * PB_HT + 8 * n + 2 * t) = make_float2(l[n][0], l[n][1]);
            }
            if (pb_bar_any(bad)) { bad = true; break; }
            const bool whole = begun_at_zero && row_ends;
            const pb_i64 part = (pb_i64)blockIdx.x * 2 + (segment ? 1 : 0);
#pragma unroll
            for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int head = 8 * n + 2 * t + e;
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; ++w) sum += wsum[w * PB_HT + head];
                    if (head >= hg) continue;
                    const pb_i64 global = (pb_i64)at.s * PB_H * group + head0 + head;
                    float* to = whole ? out + global * PB_D : partial + (part * PB_HT + head) * PB_D;
                    const float inv = whole ? 1.0f / sum : 1.0f;
#pragma unroll
                    for (int a = 0; a < PB_MTW; ++a) {
                        const int ch = (warp + 4 * a) * 16 + g;
                        if (ch < PB_D) to[ch] = o[a][n][e] * inv;
                        if (ch + 8 < PB_D) to[ch + 8] = o[a][n][e + 2] * inv;
                    }
                    if (warp == 0 && g == 0) {
                        if (!whole) partial_ml[part * PB_HT + head] = make_float2(m[n][e], sum);
#if PB_SCORED
                        else norms[global] = make_float2(m[n][e], 1.0f / sum);
#endif
                    }
                }
            ++segment;
        }
    }
    if (bad) abort_flag = 1;
}

// A row in several parts: {row, first CTA, number of parts, the first part's
// place}. Part i's sums for a query head.
static __device__ __forceinline__ pb_i64 pb_part(const int4& r, int i, int head) {
    return (pb_i64)(2 * (r.y + i) + (i ? 0 : r.w)) * PB_HT + head;
}

// Joins the parts of a row that several CTAs worked on. Block: one query head
// of one such row; its threads read the parts' sums at once, then each group of
// D / 4 threads takes every PB_JOIN-th part, four channels a thread, its first
// two on their way beside the sums. Latency: one round of loads.
#define PB_JOIN (PB_JOIN_THREADS / (PB_D / 4))
static __device__ __forceinline__ void pb_join(const int4* joins, const float* partial, const float2* partial_ml,
                                               float* out, int group, int chunks, int block) {
    __shared__ float weight[PB_JOIN_THREADS], reduce[16];
    __shared__ float4 sums[PB_JOIN_THREADS];
    const int heads = min(group, PB_HT);
    const int4 r = joins[block / heads]; // of the plan, in place before the launch
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int head = block % heads, chunk = r.x % chunks, kvh = (r.x / chunks) % PB_H, s = r.x / chunks / PB_H;
    if (head >= group - chunk * PB_HT) return;
    const pb_i64 global = (pb_i64)s * PB_H * group + kvh * group + chunk * PB_HT + head;
    const int lane = threadIdx.x & 31, quad = threadIdx.x % (PB_D / 4), team = threadIdx.x / (PB_D / 4);
    float top = __int_as_float(0xff800000), sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int from = 0; from < r.z; from += PB_JOIN_THREADS) { // one round unless a row has over PB_JOIN_THREADS parts
        const int n = min(PB_JOIN_THREADS, r.z - from), i = from + threadIdx.x;
        float2 ml = make_float2(__int_as_float(0xff800000), 0.0f);
        if (threadIdx.x < n) ml = partial_ml[pb_part(r, i, head)];
        float4 early[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (team < PB_JOIN && team + e * PB_JOIN < n)
                early[e] = *reinterpret_cast<const float4*>(partial + pb_part(r, from + team + e * PB_JOIN, head) * PB_D + 4 * quad);
        float x = ml.x;
#pragma unroll
        for (int m = 16; m > 0; m /= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
        __syncthreads();
        if (lane == 0) reduce[threadIdx.x >> 5] = x;
        __syncthreads();
        x = top;
#pragma unroll
        for (int w = 0; w < PB_JOIN_THREADS / 32; ++w) x = fmaxf(x, reduce[w]);
        const float corr = pb_exp2(top - x);
        top = x;
        const float w = threadIdx.x < n ? pb_exp2(ml.x - top) : 0.0f;
        weight[threadIdx.x] = w;
        float y = w * ml.y;
#pragma unroll
        for (int m = 16; m > 0; m /= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
        __syncthreads();
        if (lane == 0) reduce[threadIdx.x >> 5] = y;
        __syncthreads();
        y = 0.0f;
#pragma unroll
        for (int w2 = 0; w2 < PB_JOIN_THREADS / 32; ++w2) y += reduce[w2];
        sum = fmaf(sum, corr, y);
        acc = make_float4(acc.x * corr, acc.y * corr, acc.z * corr, acc.w * corr);
        if (team < PB_JOIN) {
            auto add = [&](const float4& o, float w) {
                acc.x = fmaf(w, o.x, acc.x);
                acc.y = fmaf(w, o.y, acc.y);
                acc.z = fmaf(w, o.z, acc.z);
                acc.w = fmaf(w, o.w, acc.w);
            };
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (team + e * PB_JOIN < n) add(early[e], weight[team + e * PB_JOIN]);
#pragma unroll 4
            for (int j = team + 2 * PB_JOIN; j < n; j += PB_JOIN)
                add(*reinterpret_cast<const float4*>(partial + pb_part(r, from + j, head) * PB_D + 4 * quad), weight[j]);
        }
    }
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (team == 0) {
        for (int w = 1; w < PB_JOIN; ++w) {
            const float4 o = sums[w * (PB_D / 4) + quad];
            acc.x += o.x;
            acc.y += o.y;
            acc.z += o.z;
            acc.w += o.w;
        }
        const float inv = 1.0f / sum;
        *reinterpret_cast<float4*>(out + global * PB_D + 4 * quad) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}

#if PB_SCORED
// new[s, h, i] = scores[s, h, i] + sum over the group of 2^(logit - top) / sum,
// where a split row's top and sum come from its parts, so that scores need not
// wait for the join. Block: 4 * PB_JOIN_THREADS slots of one sequence and key
// head, the norms of up to 64 query heads at a time in shared memory.
static __device__ __forceinline__ void pb_load_logits(float (&x)[4][4], const float* l, int heads, int i0, int length,
                                                      pb_i64 longest) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * PB_JOIN_THREADS;
            x[e][j] = e < heads && i < length ? l[e * longest + i] : 0.0f;
        }
}
static __device__ __forceinline__ void pb_scores(const int4* joins, const int* split, const float2* partial_ml,
                                                 const float* logits, const float2* norms, const int* lengths,
                                                 const float* scores, float* out, pb_i64 longest, pb_i64 ns, int group,
                                                 int chunks, pb_u32 block) {
    __shared__ float2 shared_norms[64];
    const pb_u32 blocks = (pb_u32)((longest + 4 * PB_JOIN_THREADS - 1) / (4 * PB_JOIN_THREADS));
    const pb_i64 row = block / blocks; // sequence and key head
    const int i0 = (int)(block % blocks) * (4 * PB_JOIN_THREADS) + threadIdx.x; // lengths are below 2^30
    const int length = lengths[row / PB_H];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float* before = scores + row * ns;
    float a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * PB_JOIN_THREADS;
        a[j] = i < length && i < ns ? before[i] : 0.0f;
    }
    // Blocks past the length only write zeros.
    for (int from = 0; from < group && (int)(block % blocks) * (4 * PB_JOIN_THREADS) < length; from += 64) {
        const int n = min(64, group - from);
        // The first heads' logits are on their way while the norms are formed.
        float x[4][4];
        const float* l = logits + (row * group + from) * longest;
        pb_load_logits(x, l, n, i0, length, longest);
        __syncthreads();
        for (int e = threadIdx.x >> 5; e < n; e += PB_JOIN_THREADS / 32) { // a warp for each head, a lane for each part
            const int lane = threadIdx.x & 31, g = from + e, at = split[row * chunks + g / PB_HT];
            float top = __int_as_float(0xff800000), sum = 0.0f;
            if (at < 0) {
                const float2 v = norms[row * group + g];
                top = v.x;
                sum = lane ? 0.0f : 1.0f / v.y;
            } else {
                const int4 r = joins[at];
                for (int i = lane; i < r.z; i += 32) {
                    const float2 ml = partial_ml[pb_part(r, i, g % PB_HT)];
                    const float now = fmaxf(top, ml.x);
                    sum = fmaf(sum, pb_exp2(top - now), ml.y * pb_exp2(ml.x - now));
                    top = now;
                }
            }
            float all = top;
#pragma unroll
            for (int m = 16; m > 0; m /= 2) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, m));
            sum = sum != 0.0f ? sum * pb_exp2(top - all) : 0.0f; // lanes without a part have no maximum
#pragma unroll
            for (int m = 16; m > 0; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            if (lane == 0) shared_norms[e] = make_float2(all, 1.0f / sum);
        }
        __syncthreads();
        for (int g = 0; g < n; g += 4) {
            if (g) pb_load_logits(x, l + g * longest, n - g, i0, length, longest);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (g + e < n)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (i0 + j * PB_JOIN_THREADS < length) a[j] = fmaf(pb_exp2(x[e][j] - shared_norms[g + e].x), shared_norms[g + e].y, a[j]);
        }
    }
    float* to = out + row * longest;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * PB_JOIN_THREADS;
        if (i < longest) to[i] = a[j];
    }
}
#endif

// The first `join_blocks` blocks join, the others score.
extern "C" __global__ void __launch_bounds__(PB_JOIN_THREADS) pb_paged_finish(
    const int4* joins, const int* split, const float* partial, const float2* partial_ml, float* out,
    const float* logits, const float2* norms, const int* lengths, const float* scores, float* new_scores, pb_i64 longest,
    pb_i64 ns, int group, int chunks, int join_blocks) {
    if (blockIdx.x < join_blocks) {
        pb_join(joins, partial, partial_ml, out, group, chunks, blockIdx.x);
        return;
    }
#if PB_SCORED
    pb_scores(joins, split, partial_ml, logits, norms, lengths, scores, new_scores, longest, ns, group, chunks,
              blockIdx.x - join_blocks);
#endif
}
)PB";
        }

        std::string defines(const form& f) {
            std::ostringstream os;
            os << "#define PB_H " << f.heads << "\n#define PB_D " << f.dim << "\n#define PB_PS " << f.page
               << "\n#define PB_ESZ " << f.width() << "\n#define PB_NT " << f.tiles8 << "\n#define PB_RING " << f.ring()
               << "\n#define PB_JOIN_THREADS " << f.join_threads << "\n#define PB_PER_SM " << f.per_sm()
               << "\n#define PB_STATIC " << form::kStatic << "\n#define PB_SCORED " << (f.scored ? 1 : 0) << "\n";
            if (f.stall != 0) os << "#define PB_TEST_STALL " << f.stall << "\n";
            return os.str();
        }

        std::atomic<int> g_test_stall{0};

        // The form for `group` query heads of each key head: 16 share a tile's
        // loads, 8 where 16 would leave the ring less than three units.
        form form_of(const kv_cache& c, int64_t group) {
            form f;
            f.heads = static_cast<int>(c.heads);
            f.dim = static_cast<int>(c.dim);
            f.page = static_cast<int>(c.page_size);
            f.bf16 = c.type == cache_type::bf16;
            f.tiles8 = group > 8 ? 2 : 1;
            if (f.ring() < 3) f.tiles8 = 1;
            return f;
        }

        const char kAttention[] = "pb_paged_attention";
        const char kFinish[] = "pb_paged_finish";

        op_kernel& kernel_of(const char* name, const form& f, uint32_t smem) {
            const op_key key{reinterpret_cast<int64_t>(name), f.heads, f.dim, f.page, f.bf16, f.scored, f.tiles8, f.join_threads, f.stall};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = name;
                k.source = std::string{kernel_prelude()} + defines(f) + device_source();
                k.smem = smem;
            });
        }

        // Even runs of 64-slot tiles, over all rows one after the other, where a
        // row counts as one tile more than it has, for its queries, its sums
        // and its result (32 sequences of 8 rows up to 4096 slots of 80 channels:
        // 39.4 us with tiles alone, 36.4 so). A run begins and ends inside a row at
        // most once each, so a CTA leaves at most two parts behind. Where every
        // row is short and they all fit, each has a CTA of its own instead: up
        // to kWholeRow tiles in a row take less time than the second launch
        // that joins parts (8 sequences of 4 rows of 384 slots: 8.9 us so, 11.4
        // in parts; of 512: 10.8 and 11.3; of 768: 15.1 and 11.5). A row without slots has a CTA that writes its
        // zeros, after the others.
        struct schedule {
            std::vector<int32_t> work; // per CTA: row, tile, tiles, 0
            std::vector<int32_t> join; // per row in parts: row, first CTA, parts, its place
            std::vector<int32_t> split; // per row: its entry of `join`, or -1
        };
        constexpr int64_t kWholeRow = 8;

        schedule make_schedule(const std::vector<int64_t>& lengths, int64_t heads, int64_t chunks, int64_t ctas) {
            schedule r;
            const int64_t per = heads * chunks;
            int64_t total = 0, rows = 0, most = 0;
            for (int64_t length : lengths) {
                const int64_t tiles = (length + 63) / 64;
                total += tiles * per;
                most = std::max(most, tiles);
                if (tiles != 0) rows += per;
            }
            const bool whole = most <= kWholeRow && rows <= ctas;
            // The tile, in the order of all rows, that each CTA begins with.
            std::vector<int64_t> starts;
            if (!whole) {
                const int64_t n = std::min(total, ctas);
                int64_t row_cost = 0, row_tile = 0, cut = 0; // where the row begins
                for (int64_t length : lengths) {
                    const int64_t tiles = (length + 63) / 64;
                    if (tiles == 0) continue;
                    for (int64_t j = 0; j < per; ++j) {
                        for (; cut < n; ++cut) {
                            const int64_t at = static_cast<int64_t>(static_cast<__int128>(total + rows) * cut / n) - row_cost;
                            if (at > tiles) break;
                            const int64_t tile = row_tile + std::max<int64_t>(0, at - 1);
                            if (starts.empty() || starts.back() != tile) starts.push_back(tile);
                        }
                        row_cost += tiles + 1;
                        row_tile += tiles;
                    }
                }
                starts.push_back(total);
            }
            const int64_t n = whole ? rows : static_cast<int64_t>(starts.size()) - 1;
            int64_t cta = 0, from = 0; // `from`: the row's first tile in the whole order
            auto start = [&](int64_t c) { return starts[static_cast<size_t>(c)]; };
            auto put = [](std::vector<int32_t>& to, std::initializer_list<int64_t> values) {
                for (int64_t v : values) to.push_back(static_cast<int32_t>(v));
            };
            std::vector<int32_t> empty;
            for (size_t s = 0; s < lengths.size(); ++s) {
                const int64_t tiles = (lengths[s] + 63) / 64;
                for (int64_t j = 0; j < per; ++j) {
                    const int64_t row = static_cast<int64_t>(s) * per + j;
                    r.split.push_back(-1);
                    if (tiles == 0) {
                        put(empty, {row, 0, 0, 0});
                        continue;
                    }
                    if (whole) {
                        put(r.work, {row, 0, tiles, 0});
                        continue;
                    }
                    // CTAs that begin in this row.
                    while (cta < n && start(cta) < from + tiles) {
                        put(r.work, {row, start(cta) - from, start(cta + 1) - start(cta), 0});
                        ++cta;
                    }
                    // Its first part belongs to the last CTA that begins at or before it.
                    int64_t first = cta - 1;
                    while (start(first) > from) --first;
                    const int64_t parts = cta - first;
                    if (parts > 1) {
                        r.split.back() = static_cast<int32_t>(r.join.size() / 4);
                        put(r.join, {row, first, parts, start(first) < from ? 1 : 0});
                    }
                    from += tiles;
                }
            }
            r.work.insert(r.work.end(), empty.begin(), empty.end());
            return r;
        }

    } // namespace

    std::vector<tensor> paged_attention(const tensor& q, kv_batch& batch, float scale, bool scored,
                                        const tensor* scores) {
        kv_cache& c = *batch.cache;
        const auto shape = shape_of(q);
        const int64_t n = batch.sequences();
        expect(shape.size() == 3 && shape[0] == n && shape[2] == c.dim,
               "paged_attention: q must be [sequences, q_heads, head_dim] of the batch");
        expect(shape[1] >= c.heads && shape[1] % c.heads == 0 && shape[1] <= 65536,
               "paged_attention: q_heads must be a multiple of the cache's kv_heads");
        // The kernels' logits are in units of log2.
        float scale2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
        expect(std::isfinite(scale2), "paged_attention: scale must be finite, and below 2.3e38");
        int64_t ns = 0;
        if (scores != nullptr) {
            const auto s = shape_of(*scores);
            expect(s.size() == 3 && s[0] == n && s[1] == c.heads,
                   "paged_attention_scored: scores must be [sequences, kv_heads, slots]");
            ns = s[2];
        }
        const int device = device_of(q, "paged_attention");
        expect(device == c.device && (scores == nullptr || device_of(*scores, "paged_attention_scored") == device),
               "paged_attention: operands must live on the cache's device");
        auto stream = current_stream(device);
        op_operand x = operand(q, stream, true), xs;
        if (scores != nullptr) xs = operand(*scores, stream, false);
        int heads = static_cast<int>(shape[1]), group = static_cast<int>(shape[1] / c.heads);
        form f = form_of(c, group);
        f.scored = scored;
        f.stall = g_test_stall.load(std::memory_order_relaxed);
        int chunks = f.chunks(group);
        const int64_t rows = n * c.heads * chunks;
        expect(rows < (int64_t{1} << 27), "paged_attention: too many sequences and heads");
        const batch_plan& plan = plan_of(batch, chunks, int64_t{f.per_sm()} * sm_count(device));

        op_result out = new_result(shape, device, stream);
        uint64_t results_ptr = out.ptr;
        int64_t longest = batch.longest;
        int width = static_cast<int>(batch.table_width), longest32 = static_cast<int>(longest);
        // Workspace: sums and results of split rows' parts, and for scores the
        // logits and each head's maximum and sum.
        const size_t part_heads = plan.joins == 0 ? 0 : static_cast<size_t>(plan.working) * 2 * static_cast<size_t>(8 * f.tiles8);
        const size_t parts = part_heads * static_cast<size_t>(c.dim), scored_heads = scored ? static_cast<size_t>(n * heads) : 0;
        const size_t all = parts + 2 * part_heads + (2 + static_cast<size_t>(longest)) * scored_heads;
        cuda_jit::device_buffer scratch;
        if (all != 0) scratch = allocate(device, all * sizeof(float), stream);
        uint64_t ml = address(scratch), partial = ml + 2 * part_heads * 4, norms = partial + parts * 4,
                 logits = norms + 2 * scored_heads * 4;
        uint64_t work = address(plan.data), join = work + static_cast<uint64_t>(plan.ctas) * 16, err = 0;
        op_kernel* attention = plan.ctas > 0 ? &kernel_of(kAttention, f, static_cast<uint32_t>(f.smem())) : nullptr;
        op_result os;
        int64_t blocks = plan.joins * std::min(group, 8 * f.tiles8);
        // A small block where each row has a few parts (many rows: 128 threads
        // take 5.7 us where 512 take 11.7), a large one where one row has many
        // (37 parts each: 12.5 us and 6.2).
        if (plan.most_parts > 16) f.join_threads = 512;
        int join_blocks = static_cast<int>(blocks);
        if (scored) {
            os = new_result({n, c.heads, longest}, device, stream);
            blocks += (longest + 4 * f.join_threads - 1) / (4 * f.join_threads) * n * c.heads;
        }
        expect(blocks <= 0x7fffffff, "paged_attention: too many sequences, heads and slots");
        op_kernel* finishing = blocks > 0 ? &kernel_of(kFinish, f, 0) : nullptr;
        order_read(*cuda_jit::buffer_access::state(batch.data), stream);
        if (plan.data.size_bytes() != 0) order_read(*cuda_jit::buffer_access::state(plan.data), stream);
        if (attention != nullptr) {
            (void)attention->on(device);
            check(pbrt_error_word(device, &err));
            void* params[] = {&c.map_k, &c.map_v, &x.ptr, &batch.lengths_at, &batch.tables_at, &work,
                              &out.ptr, &partial, &ml, &logits, &norms, &width, &group, &chunks,
                              &x.strides[0], &x.strides[1], &longest32, &scale2, &err};
            std::scoped_lock lock{c.order};
            order_read(*cuda_jit::buffer_access::state(c.k), stream);
            order_read(*cuda_jit::buffer_access::state(c.v), stream);
            op_launch(*attention, device, stream, {static_cast<uint32_t>(plan.ctas), 1, 1}, 160, params);
        }
        if (finishing != nullptr) {
            uint64_t split = join + static_cast<uint64_t>(plan.joins) * 16;
            void* params[] = {&join,   &split,   &partial, &ml,  &results_ptr, &logits, &norms,      &batch.lengths_at,
                              &xs.ptr, &os.ptr,  &longest, &ns,  &group,       &chunks, &join_blocks};
            op_launch(*finishing, device, stream, {static_cast<uint32_t>(blocks), 1, 1},
                      static_cast<uint32_t>(f.join_threads), params);
        }
        std::vector<tensor> results;
        results.push_back(finish(std::move(out)));
        if (scored) results.push_back(finish(std::move(os)));
        return results;
    }

    void set_test_attention_stall(int mode) { g_test_stall.store(mode); }

    std::pair<int, int> attention_shape(int64_t dim, cache_type type, int64_t group) {
        kv_cache c;
        c.dim = dim;
        c.type = type;
        const form f = form_of(c, group);
        return {f.per_sm(), f.shared()};
    }

    const batch_plan& plan_of(kv_batch& batch, int64_t chunks, int64_t ctas) {
        if (batch.plans->hint != nullptr) {
            std::scoped_lock lock{batch.plans->hint->mutex};
            batch.plans->hint->chunks = chunks;
            batch.plans->hint->ctas = ctas;
        }
        std::scoped_lock lock{batch.plans->mutex};
        for (const auto& p : batch.plans->made)
            if (p->chunks == chunks && p->limit == ctas) return *p;
        schedule s = make_schedule(batch.lengths, batch.cache->heads, chunks, ctas);
        auto p = std::make_unique<batch_plan>();
        p->chunks = chunks;
        p->limit = ctas;
        p->ctas = static_cast<int64_t>(s.work.size() / 4);
        for (size_t i = 2; i < s.work.size(); i += 4) p->working += s.work[i] != 0;
        p->joins = static_cast<int64_t>(s.join.size() / 4);
        for (size_t i = 2; i < s.join.size(); i += 4) p->most_parts = std::max<int64_t>(p->most_parts, s.join[i]);
        s.work.insert(s.work.end(), s.join.begin(), s.join.end());
        s.work.insert(s.work.end(), s.split.begin(), s.split.end());
        const int device = batch.cache->device;
        auto stream = upload_stream(device);
        p->data = allocate(device, s.work.size() * sizeof(int32_t), stream);
        check(pbrt_memcpy_h2d_async(device, address(p->data), s.work.data(), s.work.size() * sizeof(int32_t), stream->stream));
        check(pbrt_stream_synchronize(device, stream->stream));
        batch.plans->made.push_back(std::move(p));
        return *batch.plans->made.back();
    }

    void prepare_plan(kv_batch& batch) {
        int64_t chunks = 0, ctas = 0;
        {
            std::scoped_lock lock{batch.plans->hint->mutex};
            chunks = batch.plans->hint->chunks;
            ctas = batch.plans->hint->ctas;
        }
        if (chunks == 0) {
            chunks = 1;
            ctas = int64_t{form_of(*batch.cache, 1).per_sm()} * sm_count(batch.cache->device);
        }
        (void)plan_of(batch, chunks, ctas);
    }

    std::string attention_schedule(const std::vector<int64_t>& lengths, int64_t heads, int64_t chunks, int64_t ctas) {
        const schedule s = make_schedule(lengths, heads, chunks, ctas);
        std::ostringstream os;
        for (size_t i = 0; i < s.work.size(); i += 4)
            os << "work " << s.work[i] << " " << s.work[i + 1] << " " << s.work[i + 2] << "\n";
        for (size_t i = 0; i < s.join.size(); i += 4)
            os << "join " << s.join[i] << " " << s.join[i + 1] << " " << s.join[i + 2] << " " << s.join[i + 3] << "\n";
        return os.str();
    }

    void paged_attention_sources(kernel_list& out) {
        for (const auto& [dim, width, tiles8, page] :
             {std::array<int, 4>{128, 2, 1, 64}, std::array<int, 4>{64, 2, 1, 16}, std::array<int, 4>{64, 4, 1, 16},
              std::array<int, 4>{128, 4, 1, 8}, std::array<int, 4>{256, 4, 1, 256}, std::array<int, 4>{256, 2, 2, 32},
              std::array<int, 4>{72, 2, 2, 32}, std::array<int, 4>{8, 4, 2, 32}}) {
            form f;
            f.heads = 8;
            f.dim = dim;
            f.bf16 = width == 2;
            f.tiles8 = tiles8;
            f.page = page;
            f.scored = true;
            out.emplace_back("pb_paged_attention_" + std::to_string(dim) + (f.bf16 ? "_bf16_" : "_f32_") + std::to_string(8 * tiles8),
                             std::string{kernel_prelude()} + defines(f) + device_source());
        }
    }

} // namespace porch::detail
