// Attention of one new token per sequence over a paged cache:
//   o = softmax(scale q K^T) V
// over the slots in use, query heads sharing key heads in groups, and its
// scored form, which adds each slot's attention weight, summed over the query
// heads of its key head, to running scores (what eviction ranks slots by).
// A sequence without slots gives zeros.
//
// Bound: HBM, which has to deliver every key and value in use once (2 x slots
// x kv_heads x head_dim x 1, 2 or 4 bytes, and 4 for the scale of an 8-bit row).
// 48 sequences up to 8191 slots, 32 query heads over 8 of 128 bfloat16 channels:
// 784 MB in 127 us = 6.2 TB/s; one sequence of 262147 slots: 1074 MB in 171 us =
// 6.3 TB/s. The same in 8 bits: 404 MB in 76 us and 554 MB in 100, 5.3 and 5.5 TB/s
// with both launches (a call, inputs rotated past the L2 cache). Scored, the 48 take
// 152 us in bfloat16 and 94 in 8 bits. Few or short rows are bound by the
// launch and the first loads' latency instead (about 6 us, 3 of the stream where
// calls follow each other).
//
// pb_paged_attention, 160 threads: a producer warp loads tiles of 64 slots (128 of
// an 8-bit cache of up to 128 channels), K then V, through a ring of TMA boxes (a
// page, or 64 rows of a larger one; 128 bytes wide, swizzled, zeros past the head
// size), and four computing warps keep an online softmax over them: S^T = K Q^T for
// 16 slots of each 64 a warp, a maximum
// over the tile, weights to shared memory, O^T += V^T P^T for a quarter of the
// channels each. The transposed products put slots and channels on the tensor
// core's 16 rows and query heads on its 8 columns, so 1 to 8 heads cost the
// same. One query per sequence and head leaves nothing for the 128-row tiles of
// tcgen05; with mma.sync the tensor pipe is 31 % busy at full bandwidth.
//
// Accuracy: float32. Queries and weights are split into three bfloat16 terms
// (24 bits) against a bfloat16 cache, whose products are then exact; a float32
// cache is split into two tf32 terms like the queries (each off by up to 2^-21,
// and of four products the smallest is left out: 2^-19.6 of a product at most).
// The tensor core's accumulator cuts low bits at every addition, so a tile's
// products start from zero and are added to the running sums in fp32, rounded to
// nearest. An 8-bit cache is multiplied as it is: queries and weights are three
// digits to base 256 of a whole number, whose sums of products are exact, and a
// slot's scales go into its score and its weight. Whole numbers have one unit for a
// head's query, 2^-22 of its largest channel, and one for a tile's weights, 2^-22 of
// its largest weight x value scale: what lies far below those has fewer bits than a
// float32 of its own would, and the result is within the other caches' 4e-7 of the
// largest that goes into it.
//
// Sequences that share a prefix (a prompt, say) read it once: their queries, up to
// 16 for one key head here, or up to 128 where the large tiles of tcgen05 pay, are
// one row over the prefix, and each has another over what follows; a last launch
// joins them. The rule, with what both sides take, is beside worth_sharing.
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

        // Slots of a tile: 128 of an 8-bit cache, whose 64 take hardly more time than
        // what a tile takes by itself (48 sequences up to 8191 slots: 78 us with 64, 72
        // so; one of 262147: 103 and 93), as long as that leaves room for several CTAs.
        int tile_of(cache_type type, int64_t dim) { return type == cache_type::i8 && dim <= 128 ? 128 : 64; }

        // The whole layout of a kernel follows from these.
        struct form {
            int heads = 1, dim = 0, page = 0;
            cache_type type = cache_type::f32;
            bool scored = false, shared = false;
            int stall = 0; // the test hook's mode
            int join_threads = 128;
            int tiles8 = 1; // groups of 8 query heads that a row holds (1 or 2)
            int width() const { return type == cache_type::f32 ? 4 : (type == cache_type::bf16 ? 2 : 1); }
            int planes() const { return (dim * width() + 127) / 128; }
            int tile() const { return tile_of(type, dim); }                    // slots
            int unit() const { return planes() * tile() * 128; }               // a tile of K or of V
            int steps() const { return ((dim * width() + 31) / 32 + 1) & ~1; } // 32-byte k-steps, an even number
            int scales() const { return type == cache_type::i8 ? tile() * 4 : 0; } // bytes of a unit's
            int terms() const { return type == cache_type::f32 ? 2 : 3; }
            int q_row() const { return steps() * 32 + 16; }
            int p_row() const { return tile() * width() + 16; }
            int small() const { // everything but the ring
                return terms() * tiles8 * 8 * (q_row() + p_row()) + 2 * 4 * tiles8 * 8 * 4 +
                       (type == cache_type::i8 ? 5 * tiles8 * 8 * 4 : 0);
            }
            int per_sm() const { return choose().first; }
            int ring() const { return choose().second; }
            int chunks(int group) const { return (group + 8 * tiles8 - 1) / (8 * tiles8); } // rows of a key head
            int smem() const { return 1024 + ring() * (unit() + scales()) + small(); }
            // What a CTA takes of an SM's 228 KB: that, the kernel's static
            // arrays (the ring's barriers and a flag, which the kernel checks
            // against kStatic) with the rounding of the sum, and the KB that
            // the system keeps for each CTA.
            static constexpr int kStatic = 256;
            int shared_bytes() const { return smem() + kStatic + 1024; }

          private:
            // CTAs of an SM and units of a CTA's ring: as many CTAs as leave
            // room for three units each, so that one is on its way while two
            // are read. CTAs hide each other's barriers (48 sequences up to
            // 8191 slots, 128 bfloat16 channels: 134 us with two CTAs of six
            // units, 124 with three of three).
            std::pair<int, int> choose() const {
                for (int n = 4; n > 1; --n) {
                    const int r = ((228 * 1024) / n - 2048 - kStatic - small()) / (unit() + scales());
                    if (r >= 3) return {n, std::min(r, 6)};
                }
                return {1, std::min((227 * 1024 - 1024 - kStatic - small()) / (unit() + scales()), 6)};
            }
        };

        const char* device_source() {
            return R"PB(
typedef long long pb_i64;
#define PB_WAIT_CYCLES 4000000000ll
#define PB_HT (8 * PB_NT)                // query heads of a row, padded
#define PB_PLANES ((PB_D * PB_ESZ + 127) / 128)
#define PB_PLANE (PB_TS * 128)
#define PB_UNIT (PB_PLANES * PB_PLANE)   // a tile's slots, one 128-byte plane after the other
#define PB_MB (PB_TS / 64)               // 16 slots of each warp
#define PB_CE (128 / PB_ESZ)             // values of a plane's row
#define PB_BOX (PB_PS < 64 ? PB_PS : 64) // slots of one tile load
#define PB_STEPS ((((PB_D * PB_ESZ + 31) / 32) + 1) & ~1)
#define PB_QROW (PB_STEPS * 32 + 16)
#define PB_PROW (PB_TS * PB_ESZ + 16)
#define PB_MT ((PB_D + 15) / 16)         // 16-channel tiles of the result
#define PB_MTW ((PB_MT + 3) / 4)         // of one warp
#if PB_ESZ == 4
#define PB_TERMS 2
#else
#define PB_TERMS 3
#endif
#if PB_ESZ == 1 // sums of products of integers are exact
typedef int pb_acc;
#else
typedef float pb_acc;
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
#if PB_ESZ == 1
// PB_BOX scales, 32 bytes or more.
static __device__ __forceinline__ void pb_bulk_load(pb_u32 dst, const float* src, pb_u32 bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"((unsigned long long)src), "r"(PB_BOX * 4), "r"(bar) : "memory");
}
static __device__ __forceinline__ float pb_shared(pb_u32 at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
#endif
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
#if PB_ESZ == 1
static __device__ __forceinline__ void pb_mma(int* c, const pb_u32* a, const pb_u32* b) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Digits of a whole number of up to PB_DIGITS = 127 (65536 + 256 + 1), base 256
// and from -127 or -128 to 127, lowest first, in its bytes: adding 128 at each
// place and flipping each byte's top bit makes the carries.
#define PB_DIGITS 8355711
#define PB_WEIGHTS 8347552.0f // of those less 2^-10
static __device__ __forceinline__ pb_u32 pb_digits(int x) { return ((pb_u32)x + 0x00808080u) ^ 0x00808080u; }
// What they say of a sum of products: exact in integers but for the last step.
static __device__ __forceinline__ float pb_of_digits(int lowest, int middle, int highest) {
    return fmaf((float)highest, 65536.0f, (float)(middle * 256 + lowest));
}
static __device__ __forceinline__ float pb_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
static __device__ __forceinline__ float pb_log2(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
#elif PB_ESZ == 2
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
// heads), tiles PB_TS slots of a row; a CTA works through a run of tiles.
#if PB_SHARED
// Sequences that share a prefix: a row is a run of slots of one key head, the
// prefix or what follows it, and the queries that read it, of sequence after
// sequence from `first` on, from the f0-th of their heads.
struct pb_at { int row, tile; int s, h, begin, length, tiles, first, f0, count; };
static __device__ __forceinline__ void pb_enter(pb_at& a, const int* rows, int) {
    const int4 x = reinterpret_cast<const int4*>(rows)[2 * a.row], y = reinterpret_cast<const int4*>(rows)[2 * a.row + 1];
    a.s = x.x;
    a.h = x.y;
    a.begin = x.z;
    a.length = x.w;
    a.first = y.x;
    a.f0 = y.y;
    a.count = y.z;
    a.tiles = (a.length - a.begin + PB_TS - 1) / PB_TS;
}
static __device__ __forceinline__ int pb_base(const pb_at& a) { return a.begin + a.tile * PB_TS; }
static __device__ __forceinline__ int pb_heads(const pb_at& a, int) { return a.count; }
static __device__ __forceinline__ pb_i64 pb_query(const pb_at& a, int head, int group, pb_i64 q_seq, pb_i64 q_head) {
    const int f = a.f0 + head;
    return (a.first + f / group) * q_seq + (a.h * group + f % group) * q_head;
}
#else
struct pb_at { int row, tile; int s, h, chunk, length, tiles; };
static __device__ __forceinline__ int pb_base(const pb_at& a) { return a.tile * PB_TS; }
static __device__ __forceinline__ int pb_heads(const pb_at& a, int group) { return min(PB_HT, group - a.chunk * PB_HT); }
static __device__ __forceinline__ pb_i64 pb_query(const pb_at& a, int head, int group, pb_i64 q_seq, pb_i64 q_head) {
    return a.s * q_seq + (a.h * group + a.chunk * PB_HT + head) * q_head;
}
static __device__ __forceinline__ void pb_enter(pb_at& a, const int* lengths, int chunks) {
    a.chunk = a.row % chunks;
    a.h = (a.row / chunks) % PB_H;
    a.s = a.row / chunks / PB_H;
    a.length = lengths[a.s];
    a.tiles = (a.length + PB_TS - 1) / PB_TS;
}
#endif
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
    const int first = pb_base(a) + lane * PB_BOX;
    return lane * PB_BOX < PB_TS && first < a.length ? tables[(pb_i64)a.s * width + first / PB_PS] : 0;
}

// A row's queries, PB_Q_EACH values of each of 128 threads, every load before
// the first use; zero past its heads and the head size.
#define PB_Q_HEAD (PB_STEPS * 32 / PB_ESZ)
#define PB_Q_EACH ((PB_HT * PB_Q_HEAD + 127) / 128)
#if PB_ESZ == 1
#define PB_Q_RUNS ((PB_Q_HEAD + 127) / 128)
#define PB_Q_EACH8 (PB_HT / 4 * PB_Q_RUNS * 4)
struct pb_queries { float x[PB_Q_EACH8]; };
#else
#define PB_Q_EACH8 PB_Q_EACH
struct pb_queries { float x[PB_Q_EACH]; };
#endif
static __device__ __forceinline__ void pb_load_queries(pb_queries& r, const float* q, const pb_at& a, pb_i64 q_seq,
                                                       pb_i64 q_head, int group) {
    const int heads = pb_heads(a, group);
#if PB_ESZ == 1 // a warp has every fourth head, a lane runs of four channels
#pragma unroll
    for (int j = 0; j < PB_Q_EACH8; ++j) {
        const int head = (threadIdx.x >> 5) + 4 * (j / (4 * PB_Q_RUNS));
        const int d = (j / 4 % PB_Q_RUNS) * 128 + (threadIdx.x & 31) * 4 + j % 4;
        r.x[j] = head < heads && d < PB_D ? __ldg(q + pb_query(a, head, group, q_seq, q_head) + d) : 0.0f;
    }
#else
#pragma unroll
    for (int j = 0; j < PB_Q_EACH; ++j) {
        const int e = threadIdx.x + 128 * j, head = e / PB_Q_HEAD, d = e % PB_Q_HEAD;
        r.x[j] = head < heads && d < PB_D ? __ldg(q + pb_query(a, head, group, q_seq, q_head) + d) : 0.0f;
    }
#endif
}
#if PB_ESZ == 1
// A head's queries as three digits each, in units of a power of two 2^-22 to
// 2^-23 of the head's largest size: 24 bits of that, and a rounding to nearest.
// A head that nowhere reaches 2^-100 counts as zeros; one that is not finite has
// a unit of NaN. Channels past the head size are zeros.
static __device__ __forceinline__ void pb_split_queries(const pb_queries& r, pb_u32 qs, float* units) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < PB_HT / 4; ++i) {
        const int head = warp + 4 * i;
        pb_u32 most = 0;
#pragma unroll
        for (int j = 0; j < 4 * PB_Q_RUNS; ++j) most = max(most, __float_as_uint(r.x[4 * PB_Q_RUNS * i + j]) & 0x7fffffffu);
#pragma unroll
        for (int m = 16; m > 0; m /= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, m));
        const bool finite = most < 0x7f800000u, zero = most < 0x0d800000u; // 2^-100
        pb_u32 power = 127 + 22 + 127 - (most >> 23); // biased
        if (finite && !zero && __uint_as_float(most) * __uint_as_float(power << 23) > (float)PB_DIGITS) --power;
        const float to = finite && !zero ? __uint_as_float(power << 23) : 0.0f;
        if (lane == 0) units[head] = finite ? (zero ? 0.0f : __uint_as_float((254 - power) << 23)) : __int_as_float(0x7fffffff);
#pragma unroll
        for (int run = 0; run < PB_Q_RUNS; ++run) {
            pb_u32 d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = pb_digits(__float2int_rn(r.x[4 * (PB_Q_RUNS * i + run) + e] * to));
            const pb_u32 low = __byte_perm(d[0], d[1], 0x5140), high = __byte_perm(d[2], d[3], 0x5140); // bytes 0 and 1 of both
            const pb_u32 tops = __byte_perm(__byte_perm(d[0], d[1], 0x0062), __byte_perm(d[2], d[3], 0x0062), 0x5410);
            const int at = run * 128 + lane * 4;
            if (at < PB_Q_HEAD) {
                const pb_u32 row = qs + head * PB_QROW + at;
                asm volatile("st.shared.u32 [%0], %1;" :: "r"(row), "r"(__byte_perm(low, high, 0x5410)) : "memory");
                asm volatile("st.shared.u32 [%0], %1;" :: "r"(row + PB_HT * PB_QROW), "r"(__byte_perm(low, high, 0x7632)) : "memory");
                asm volatile("st.shared.u32 [%0], %1;" :: "r"(row + 2 * PB_HT * PB_QROW), "r"(tops) : "memory");
            }
        }
    }
}
#endif

extern "C" __global__ void __launch_bounds__(160, PB_PER_SM) pb_paged_attention(
    const __grid_constant__ pb_tmap map_k, const __grid_constant__ pb_tmap map_v, const float* q, const int* lengths,
    const int* tables, const int4* work, float* out, float* partial, float2* partial_ml, float* logits, float2* norms,
    int width, int group, int chunks, pb_i64 q_seq, pb_i64 q_head, int longest, float scale2, int* err,
    const float* scales_k, const float* scales_v) {
    extern __shared__ char raw[];
    __shared__ pb_u64 bars[2 * PB_RING];
    __shared__ int abort_flag;
    static_assert(sizeof(bars) + sizeof(abort_flag) + 128 <= PB_STATIC, "shared memory that the launch does not count");
    const pb_u32 ring = (pb_smem(raw) + 1023u) & ~1023u;
    const pb_u32 unit_scales = ring + PB_RING * PB_UNIT; // of each unit, in 8 bits
    const pb_u32 qs = unit_scales + (PB_ESZ == 1 ? PB_RING * PB_TS * 4 : 0);
    const pb_u32 ps = qs + PB_TERMS * PB_HT * PB_QROW;
    float* wmax = reinterpret_cast<float*>(raw + (ps + PB_TERMS * PB_HT * PB_PROW - pb_smem(raw)));
    float* wsum = wmax + 4 * PB_HT;
#if PB_ESZ == 1
    float* wscaled = wsum + 4 * PB_HT; // the warps' maxima of weight x value scale, in log2 and relative to wmax
    float* units = wscaled + 4 * PB_HT; // of the row's queries
#endif
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
            const int base = pb_base(at), boxes = (min(PB_TS, at.length - base) + PB_BOX - 1) / PB_BOX;
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
                if (lane == 0) pb_mbar_expect_tx(full + 8 * slot, boxes * PB_BOX * (128 * PB_PLANES + (PB_ESZ == 1 ? 4 : 0)));
                __syncwarp();
                if (lane < boxes) {
                    const pb_u32 dst = ring + slot * PB_UNIT + lane * PB_BOX * 128;
#pragma unroll
                    for (int c = 0; c < PB_PLANES; ++c)
                        pb_tma_load(dst + c * PB_PLANE, which ? &map_v : &map_k, full + 8 * slot, c * PB_CE, y);
#if PB_ESZ == 1
                    pb_bulk_load(unit_scales + slot * (PB_TS * 4) + lane * PB_BOX * 4, (which ? scales_v : scales_k) + y, full + 8 * slot);
#endif
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
        for (int e = threadIdx.x; e < pb_heads(at, group) * PB_D; e += 128)
            out[pb_query(at, e / PB_D, group, PB_H * group, 1) * PB_D + e % PB_D] = 0.0f;
        return;
    }
    const int g = lane >> 2, t = lane & 3;
    int slot = 0;
    pb_u32 parity = 0;
    bool bad = false, fresh = true;
    int segment = 0; // how many rows this CTA has begun
    float m[PB_NT][2], l[PB_NT][2], o[PB_MTW][PB_NT][4];
    bool begun_at_zero = true;
#if PB_ESZ == 1
    float query_unit[PB_NT][2];
#elif PB_ESZ == 4
    // Where this thread's four values of V^T lie in each of its channel tiles
    // (slots 2 t and 2 t + 1 of a group of 8, channels g and g + 8).
    pb_u32 v_at[PB_MTW][4];
#pragma unroll
    for (int a = 0; a < PB_MTW; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 2 * t + (e >> 1), ch = (warp + 4 * a) * 16 + g + (e & 1) * 8;
            v_at[a][e] = (ch >> 5) * PB_PLANE + r * 128 + ((((ch & 31) >> 2) ^ r) << 4) + (ch & 3) * 4;
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
        const int hg = pb_heads(at, group); // query heads of this row
        if (fresh) {
            begun_at_zero = at.tile == 0;
            // The row's queries, split into terms; zero past the head size.
            if (PB_Q_EACH8 > 8 && i) pb_load_queries(ahead, q, at, q_seq, q_head, group);
#if PB_ESZ == 1
            pb_split_queries(ahead, qs, units);
#else
#pragma unroll
            for (int j = 0; j < PB_Q_EACH; ++j) {
                const int e = threadIdx.x + 128 * j, head = e / PB_Q_HEAD, d = e % PB_Q_HEAD;
                if (e < PB_HT * PB_Q_HEAD) pb_split_store(qs + head * PB_QROW + d * PB_ESZ, PB_HT * PB_QROW, ahead.x[j]);
            }
#endif
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
#if PB_ESZ == 1
#pragma unroll
            for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) query_unit[n][e] = units[8 * n + 2 * t + e] * scale2;
#endif
        }
        if (PB_Q_EACH8 <= 8 && i + 1 < mine.z && next_fresh) pb_load_queries(ahead, q, next, q_seq, q_head, group);
        const int base = pb_base(at), valid = min(PB_TS, at.length - base);

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
        pb_acc c[PB_MB][PB_TERMS + 1][PB_NT][4];
#pragma unroll
        for (int b = 0; b < PB_MB; ++b)
#pragma unroll
            for (int x = 0; x < PB_TERMS + 1; ++x)
#pragma unroll
                for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[b][x][n][e] = 0;
        {
            const int r = 16 * warp + (lane & 15);
            const pb_u32 krow = ring + slot * PB_UNIT + r * 128;
            const pb_u32 qrow = qs + (lane & 7) * PB_QROW + (lane >> 3) * 16;
#pragma unroll
            for (int k2 = 0; k2 < PB_STEPS / 2; ++k2) {
                pb_u32 slots[PB_MB][2][4]; // of 64 b + 16 warp and following
#pragma unroll
                for (int b = 0; b < PB_MB; ++b)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int chunk = (2 * k2 + k) * 2; // 16-byte chunk of the row; its plane and place
                        pb_ldm4(slots[b][k], krow + b * 8192 + (chunk >> 3) * PB_PLANE + ((((chunk & 7) + (lane >> 4)) ^ (r & 7)) << 4));
                    }
                pb_u32 (&a)[2][4] = slots[0];
#if PB_ESZ == 1
#pragma unroll
                for (int x = 0; x < PB_TERMS; ++x)
#pragma unroll
                    for (int n = 0; n < PB_NT; ++n) {
                        pb_u32 b[4];
                        pb_ldm4(b, qrow + (x * PB_HT + n * 8) * PB_QROW + k2 * 64);
#pragma unroll
                        for (int i = 0; i < PB_MB; ++i) {
                            pb_mma(c[i][x][n], slots[i][0], b);
                            pb_mma(c[i][x][n], slots[i][1], b + 2);
                        }
                    }
#elif PB_ESZ == 2
#pragma unroll
                for (int x = 0; x < PB_TERMS; ++x)
#pragma unroll
                    for (int n = 0; n < PB_NT; ++n) {
                        pb_u32 b[4];
                        pb_ldm4(b, qrow + (x * PB_HT + n * 8) * PB_QROW + k2 * 64);
                        pb_mma(c[0][x][n], a[0], b);
                        pb_mma(c[0][x == 0 ? PB_TERMS : x][n], a[1], b + 2);
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
                    pb_mma(c[0][0][n], hi[0], b);
                    pb_mma(c[0][1][n], hi[0], b2);
                    pb_mma(c[0][PB_TERMS][n], hi[1], b + 2);
                    pb_mma(c[0][1][n], lo[0], b);
                    pb_mma(c[0][1][n], hi[1], b2 + 2);
                    pb_mma(c[0][1][n], lo[1], b + 2);
                }
#endif
            }
        }
#if PB_ESZ == 1
        // The scales of this thread's slots, 0 past the sequence's end.
        float key_scale[PB_MB][2], value_scale[PB_MB][2];
        auto scale_of = [&](int i) { return i < valid ? pb_shared(unit_scales + slot * (PB_TS * 4) + i * 4) : 0.0f; };
#pragma unroll
        for (int b = 0; b < PB_MB; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) key_scale[b][j] = scale_of(64 * b + 16 * warp + g + 8 * j);
#endif
        __syncwarp();
        // Not after a wait that gave up: the unit's load may still be on its
        // way, and the producer would issue another one into it.
        if (lane == 0 && !bad) pb_mbar_arrive(empty + 8 * slot);
        if (++slot == PB_RING) { slot = 0; parity ^= 1u; }

        auto wait_for_values = [&] { bad |= !pb_wait(full + 8 * slot, parity, &abort_flag, err, 4); };

        // Logits in units of log2, -inf past the sequence's end. Thread: slots
        // 16 warp + g and + 8 (of each 64), heads 8 n + 2 t and + 1.
        float s[PB_MB][PB_NT][4], top[PB_NT][2];
#pragma unroll
        for (int n = 0; n < PB_NT; ++n) {
#pragma unroll
            for (int b = 0; b < PB_MB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at_slot = 64 * b + 16 * warp + g + (e >> 1) * 8;
#if PB_ESZ == 1
                    const float x = pb_of_digits(c[b][0][n][e], c[b][1][n][e], c[b][2][n][e]) * query_unit[n][e & 1] * key_scale[b][e >> 1];
#elif PB_TERMS == 3
                    const float x = (c[b][2][n][e] + c[b][1][n][e] + (c[b][0][n][e] + c[b][3][n][e])) * scale2;
#else
                    const float x = (c[b][1][n][e] + (c[b][0][n][e] + c[b][2][n][e])) * scale2;
#endif
                    s[b][n][e] = at_slot < valid ? x : __int_as_float(0xff800000);
#if PB_SCORED
                    const int head = 8 * n + 2 * t + (e & 1);
                    if (at_slot < valid && head < hg)
                        logits[pb_query(at, head, group, PB_H * group, 1) * longest + base + at_slot] = x;
#endif
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(s[0][n][e], s[0][n][e + 2]);
#pragma unroll
                for (int b = 1; b < PB_MB; ++b) x = fmaxf(x, fmaxf(s[b][n][e], s[b][n][e + 2]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                top[n][e] = PB_ESZ == 1 ? fmaxf(x, PB_LOWEST) : x; // 8 bits: logits are taken relative to it
            }
            if (g == 0) *reinterpret_cast<float2*>(wmax + warp * PB_HT + 8 * n + 2 * t) = make_float2(top[n][0], top[n][1]);
        }
#if PB_ESZ == 1
        wait_for_values(); // earlier than in other types: their scales go into the weights
        float scaled[PB_MB][2];
#pragma unroll
        for (int b = 0; b < PB_MB; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                value_scale[b][j] = scale_of(64 * b + 16 * warp + g + 8 * j);
                scaled[b][j] = pb_log2(value_scale[b][j]);
            }
#pragma unroll
        for (int n = 0; n < PB_NT; ++n) {
            float2 most;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = PB_LOWEST;
#pragma unroll
                for (int b = 0; b < PB_MB; ++b)
                    x = pb_max_nan(x, pb_max_nan((s[b][n][e] - top[n][e]) + scaled[b][0], (s[b][n][e + 2] - top[n][e]) + scaled[b][1]));
                x = pb_max_nan(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = pb_max_nan(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = pb_max_nan(x, __shfl_xor_sync(0xffffffffu, x, 16));
                if (e) most.y = x; else most.x = x;
            }
            if (g == 0) *reinterpret_cast<float2*>(wscaled + warp * PB_HT + 8 * n + 2 * t) = most;
        }
#endif
        if (pb_bar_any(bad)) { bad = true; break; }

        // ---- weights relative to the running maximum, split into terms
        float corr[PB_NT][2];
#if PB_ESZ == 1
        // weight x value scale, in units of which a tile's largest is up to
        // PB_DIGITS (but for 2^-10 of it, what its logarithms may be off by) and
        // at least half that; the unit is 2^power of the weights' over that.
        // Logits are taken relative to a warp's maximum before the scale's logarithm
        // is added, and the warp's to the running one after that: such a difference
        // is exact where the two lie within a factor of two, and otherwise matters
        // only up to some 2^9 (beyond, weight x scale is below 2^-100), so whatever
        // size logits have, five sums are off by 2^-16 each at most, lg2 by 2^-15 and
        // the weight's own exponent by 2^-16: 2^-13.7 of the weight. (Adding the
        // logarithm to the logit itself rounded it at the logit's size, and from 2^15
        // on a weight could pass PB_DIGITS and come out negative.)
        float power[PB_NT][2];
#endif
#pragma unroll
        for (int n = 0; n < PB_NT; ++n) {
            float2 x[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                x[w] = *reinterpret_cast<const float2*>(wmax + w * PB_HT + 8 * n + 2 * t);
                top[n][0] = fmaxf(top[n][0], x[w].x);
                top[n][1] = fmaxf(top[n][1], x[w].y);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float now = fmaxf(m[n][e], top[n][e]);
                corr[n][e] = pb_exp2(m[n][e] - now);
                m[n][e] = now;
                l[n][e] *= corr[n][e];
#if PB_ESZ == 1
                float most = PB_LOWEST;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    most = pb_max_nan(most, wscaled[w * PB_HT + 8 * n + 2 * t + e] + ((e ? x[w].y : x[w].x) - now));
                // What lies 2^-100 below the running maximum's weight weighs nothing.
                power[n][e] = pb_max_nan(ceilf(most), -100.0f);
#endif
            }
#pragma unroll
            for (int b = 0; b < PB_MB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = pb_exp2(s[b][n][e] - m[n][e & 1]);
                    l[n][e & 1] += p;
                    const int at_slot = 64 * b + 16 * warp + g + (e >> 1) * 8, head = 8 * n + 2 * t + (e & 1);
#if PB_ESZ == 1
                    // As V's fragments count slots: 2 t, 2 t + 1, 2 t + 8, 2 t + 9 side by side.
                    const int place = (at_slot & ~15) + ((at_slot & 7) >> 1) * 4 + ((at_slot >> 3) & 1) * 2 + (at_slot & 1);
                    const pb_u32 digits = pb_digits(__float2int_rn(p * value_scale[b][e >> 1] * (pb_exp2(-power[n][e & 1]) * PB_WEIGHTS)));
                    const pb_u32 to = ps + head * PB_PROW + place;
                    asm volatile("st.shared.u8 [%0], %1;" :: "r"(to), "r"(digits) : "memory");
                    asm volatile("st.shared.u8 [%0], %1;" :: "r"(to + PB_HT * PB_PROW), "r"(digits >> 8) : "memory");
                    asm volatile("st.shared.u8 [%0], %1;" :: "r"(to + 2 * PB_HT * PB_PROW), "r"(digits >> 16) : "memory");
#else
#if PB_ESZ == 2
                    const int place = at_slot;
#else
                    const int place = (at_slot & ~7) + ((at_slot & 7) >> 1) + (at_slot & 1) * 4; // as V's fragments count slots
#endif
                    pb_split_store(ps + head * PB_PROW + place * PB_ESZ, PB_HT * PB_PROW, p);
#endif
                }
        }
#if PB_ESZ != 1
        wait_for_values();
#endif
        if (pb_bar_any(bad)) { bad = true; break; }

        // ---- O^T += V^T P^T: this warp's channels x all heads. The tile's sum
        // starts from zero in the tensor core, whose additions cut low bits,
        // and is added to the running one in fp32, rounded to nearest.
        {
            const pb_u32 vunit = ring + slot * PB_UNIT;
            const pb_u32 prow = ps + (lane & 7) * PB_PROW + (lane >> 3) * 16;
            pb_acc d[PB_MTW][PB_NT][PB_ESZ == 1 ? 3 : 2][4];
#pragma unroll
            for (int a = 0; a < PB_MTW; ++a)
#pragma unroll
                for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                    for (int x = 0; x < (PB_ESZ == 1 ? 3 : 2); ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[a][n][x][e] = 0;
#pragma unroll
            for (int k2 = 0; k2 < PB_ESZ * PB_MB; ++k2) { // two k-steps at a time
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
#if PB_ESZ == 1
                            // Transposed as pairs of bytes: a register has channels 2 g and
                            // 2 g + 1 of two slots; rows g and g + 8 of the product are
                            // those two, and its columns the slots as they come. What
                            // lies past the end is finite, and its weight 0.
                            const int r = (2 * k2 + k) * 32 + lane;
                            pb_u32 pair[4];
                            pb_ldm4t(pair, vunit + (mt >> 3) * PB_PLANE + r * 128 + (((mt & 7) ^ (r & 7)) << 4));
                            v[0] = __byte_perm(pair[0], pair[1], 0x6420);
                            v[1] = __byte_perm(pair[0], pair[1], 0x7531);
                            v[2] = __byte_perm(pair[2], pair[3], 0x6420);
                            v[3] = __byte_perm(pair[2], pair[3], 0x7531);
#pragma unroll
                            for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                                for (int x = 0; x < 3; ++x) pb_mma(d[a][n][x], v, b[x][n] + 2 * k);
#elif PB_ESZ == 2
                            const int first = (2 * k2 + k) * 16;
                            const int r = first + (lane >> 4) * 8 + (lane & 7);
                            const int chunk = mt * 2 + ((lane >> 3) & 1);
                            pb_ldm4t(v, vunit + (chunk >> 3) * PB_PLANE + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
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
#if PB_ESZ == 1
                        o[a][n][e] = fmaf(pb_of_digits(d[a][n][0][e], d[a][n][1][e], d[a][n][2][e]),
                                          pb_exp2(power[n][e & 1]) * (1.0f / PB_WEIGHTS), o[a][n][e] * corr[n][e & 1]);
#else
                        o[a][n][e] = fmaf(o[a][n][e], corr[n][e & 1], d[a][n][1][e] + d[a][n][0][e]);
#endif
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
            const bool whole = !PB_SHARED && begun_at_zero && row_ends;
#if PB_SHARED
            const pb_i64 part = (pb_i64)mine.w + segment;
#else
            const pb_i64 part = (pb_i64)blockIdx.x * 2 + (segment ? 1 : 0);
#endif
#pragma unroll
            for (int n = 0; n < PB_NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int head = 8 * n + 2 * t + e;
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; ++w) sum += wsum[w * PB_HT + head];
                    if (head >= hg) continue;
                    const pb_i64 global = pb_query(at, head, group, PB_H * group, 1);
                    float* to = whole ? out + global * PB_D : partial + (part * PB_HT + head) * PB_D;
                    const float inv = whole ? 1.0f / sum : 1.0f;
#pragma unroll
                    for (int a = 0; a < PB_MTW; ++a) {
#if PB_ESZ == 1 // head sizes are whole tiles of channels
                        const int ch = (warp + 4 * a) * 16 + 2 * g;
                        if (ch < PB_D) *reinterpret_cast<float2*>(to + ch) = make_float2(o[a][n][e] * inv, o[a][n][e + 2] * inv);
#else
                        const int ch = (warp + 4 * a) * 16 + g;
                        if (ch < PB_D) to[ch] = o[a][n][e] * inv;
                        if (ch + 8 < PB_D) to[ch + 8] = o[a][n][e + 2] * inv;
#endif
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

#if PB_SHARED
// Joins the parts of a query head that reads a shared prefix and what follows
// it. Parts of a row lie one behind the other: {first, how many} of each in
// `rows`; a sequence's key head is {its first row, the prefix's first row (-1
// where there is none), its first query's place among those that read the
// prefix}. `h1`, `h2`: queries of a row of the prefix and of a sequence. A prefix's
// own stage leaves two sums for each of its queries, and results four queries of
// four channels each side by side (`own`).
//
// PB_JOIN_THREADS 32, up to 32 parts: a warp has 32 channels of four queries, the
// `units` {prefix's row or -1, first query, first sequence, key head + 2^20 x how
// many}, and every part's on the way at once, so that it reads whole lines and
// needs no barrier (64 sequences of 32 heads with 11 to 14 parts: 7 us of the
// stream, 9.8 with a warp for each query's channels, 28 with a block each).
#if PB_JOIN_THREADS == 32
#define PB_CHUNKS ((PB_D + 31) / 32)
extern "C" __global__ void __launch_bounds__(128) pb_shared_finish(
    const int4* outs, const int2* rows, const float* partial1, const float2* ml1, const float* partial2, const float2* ml2,
    float* out, int group, int h1, int h2, int own, const int4* units, int count) {
    const int lane = threadIdx.x & 31, id = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (id >= count * PB_CHUNKS) return;
    const int4 u = units[id / PB_CHUNKS]; // of the plan, in place before the launch
    const int j = lane & 3, quad = id % PB_CHUNKS * 8 + (lane >> 2), kvh = u.w & 0xfffff;
    const int f = u.y + min(j, (u.w >> 20) - 1), head = f % group, seq = u.z + f / group;
    const int4 o = outs[seq * PB_H + kvh];
    int2 r1 = make_int2(0, 0), r2 = make_int2(0, 0);
    if (u.x >= 0) r1 = rows[u.x];
    if (o.x >= 0) r2 = rows[o.x + head / h2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int parts = r1.y + r2.y;
    const int most = __reduce_max_sync(0xffffffffu, parts);
    if (most == 0) return; // already there
    // Lane (i % 8, j) has the maxima and sums of query j's parts i, i + 8, ...
    float top = PB_LOWEST, w[4], sum = 0.0f;
    float2 ml[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = 8 * k + (lane >> 2);
        ml[k] = make_float2(PB_LOWEST, 0.0f);
        if (i < r1.y) {
            const float2* p = ml1 + (pb_i64)(r1.x + i) * (1 + own) * h1 + f % h1;
            ml[k] = p[0];
            if (own) ml[k].y += p[h1].y;
        } else if (i < parts) {
            ml[k] = ml2[((pb_i64)r2.x + i - r1.y) * h2 + head % h2];
        }
        top = fmaxf(top, ml[k].x);
    }
    // Every part's results on the way; nothing of them is used before the weights are there.
    const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const bool in = quad < PB_D / 4;
    const float4* p1 = reinterpret_cast<const float4*>(partial1) + (pb_i64)r1.x * h1 * (PB_D / 4) +
                       (own ? (f % h1 / 4 * (PB_D / 4) + quad) * 4 + f % 4 : f % h1 * (PB_D / 4) + quad);
    const float4* p2 = reinterpret_cast<const float4*>(partial2) + ((pb_i64)r2.x * h2 + head % h2) * (PB_D / 4) + quad;
    auto result = [&](int i) {
        return !in || i >= parts ? none : (i < r1.y ? p1[(pb_i64)i * h1 * (PB_D / 4)] : p2[(pb_i64)(i - r1.y) * h2 * (PB_D / 4)]);
    };
    float4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = result(i);
#pragma unroll
    for (int m = 4; m < 32; m *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        w[k] = 8 * k + (lane >> 2) < parts ? pb_exp2(ml[k].x - top) : 0.0f;
        sum = fmaf(w[k], ml[k].y, sum);
    }
#pragma unroll
    for (int m = 4; m < 32; m *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    float4 acc = none;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (8 * k >= most) break;
        float4 y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = x[i];
            if (k < 3 && 8 * (k + 1) < most) x[i] = result(8 * (k + 1) + i);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = __shfl_sync(0xffffffffu, w[k], i * 4 + j);
            acc.x = fmaf(v, y[i].x, acc.x);
            acc.y = fmaf(v, y[i].y, acc.y);
            acc.z = fmaf(v, y[i].z, acc.z);
            acc.w = fmaf(v, y[i].w, acc.w);
        }
    }
    const float inv = 1.0f / sum;
    if (in && parts != 0 && j < (u.w >> 20))
        *reinterpret_cast<float4*>(out + (((pb_i64)seq * PB_H + kvh) * group + head) * PB_D + 4 * quad) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}
#else
#define PB_JOIN (PB_JOIN_THREADS / (PB_D / 4))
extern "C" __global__ void __launch_bounds__(PB_JOIN_THREADS) pb_shared_finish(
    const int4* outs, const int2* rows, const float* partial1, const float2* ml1, const float* partial2, const float2* ml2,
    float* out, int group, int h1, int h2, int own, const int4*, int) {
    __shared__ float weight[PB_JOIN_THREADS], reduce[16];
    __shared__ float4 sums[PB_JOIN_THREADS];
    const int head = blockIdx.x % group;
    const int4 o = outs[blockIdx.x / group]; // of the plan, in place before the launch
    int2 r1 = make_int2(0, 0), r2 = make_int2(0, 0);
    const int f = o.z + head;
    if (o.y >= 0) r1 = rows[o.y + f / h1];
    if (o.x >= 0) r2 = rows[o.x + head / h2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int parts = r1.y + r2.y;
    if (parts == 0) return; // already there
    const float* p1 = partial1 + (pb_i64)r1.x * h1 * PB_D + (own ? (f % h1 / 4 * PB_D + f % 4) * 4 : f % h1 * PB_D);
    const float* p2 = partial2 + ((pb_i64)r2.x * h2 + head % h2) * PB_D;
    const int lane = threadIdx.x & 31, quad = threadIdx.x % (PB_D / 4), team = threadIdx.x / (PB_D / 4);
    const int step1 = own ? 16 : 4; // from quad to quad
    auto result = [&](int i) {
        return *reinterpret_cast<const float4*>(i < r1.y ? p1 + (pb_i64)i * h1 * PB_D + quad * step1
                                                         : p2 + (pb_i64)(i - r1.y) * h2 * PB_D + quad * 4);
    };
    float top = PB_LOWEST, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int from = 0; from < parts; from += PB_JOIN_THREADS) {
        const int n = min(PB_JOIN_THREADS, parts - from), i = from + threadIdx.x;
        float2 ml = make_float2(PB_LOWEST, 0.0f);
        if (threadIdx.x < n) {
            if (i < r1.y) {
                const float2* at = ml1 + (pb_i64)(r1.x + i) * (1 + own) * h1 + f % h1;
                ml = at[0];
                if (own) ml.y += at[h1].y;
            } else {
                ml = ml2[((pb_i64)r2.x + i - r1.y) * h2 + head % h2];
            }
        }
        float4 early[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (team < PB_JOIN && team + e * PB_JOIN < n) early[e] = result(from + team + e * PB_JOIN);
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
        float y = threadIdx.x < n ? w * ml.y : 0.0f;
#pragma unroll
        for (int m = 16; m > 0; m /= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
        __syncthreads();
        if (lane == 0) reduce[threadIdx.x >> 5] = y;
        __syncthreads();
        y = 0.0f;
#pragma unroll
        for (int v = 0; v < PB_JOIN_THREADS / 32; ++v) y += reduce[v];
        sum = fmaf(sum, corr, y);
        acc = make_float4(acc.x * corr, acc.y * corr, acc.z * corr, acc.w * corr);
        if (team < PB_JOIN) {
            auto add = [&](const float4& v, float w) {
                acc.x = fmaf(w, v.x, acc.x);
                acc.y = fmaf(w, v.y, acc.y);
                acc.z = fmaf(w, v.z, acc.z);
                acc.w = fmaf(w, v.w, acc.w);
            };
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (team + e * PB_JOIN < n) add(early[e], weight[team + e * PB_JOIN]);
#pragma unroll 4
            for (int j = team + 2 * PB_JOIN; j < n; j += PB_JOIN)
                add(result(from + j), weight[j]);
        }
    }
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (team == 0) {
        for (int w = 1; w < PB_JOIN; ++w) {
            const float4 v = sums[w * (PB_D / 4) + quad];
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
        }
        const float inv = 1.0f / sum;
        *reinterpret_cast<float4*>(out + (pb_i64)blockIdx.x * PB_D + 4 * quad) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}
#endif
#else
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
    // The next launch may begin beside this one (48 sequences to 8191 slots, in 8 and in
    // 16 bits: 72.4 and 125 us a call, 72.9 and 127 where it waits for its end). After
    // pb_shared_finish that took 0.8 us longer: its next launch needs whole SMs.
    asm volatile("griddepcontrol.launch_dependents;");
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
    asm volatile("griddepcontrol.launch_dependents;");
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
#endif
)PB";
        }

        std::string defines(const form& f) {
            std::ostringstream os;
            os << "#define PB_H " << f.heads << "\n#define PB_D " << f.dim << "\n#define PB_PS " << f.page
               << "\n#define PB_ESZ " << f.width() << "\n#define PB_NT " << f.tiles8 << "\n#define PB_RING " << f.ring()
               << "\n#define PB_TS " << f.tile()
               << "\n#define PB_JOIN_THREADS " << f.join_threads << "\n#define PB_PER_SM " << f.per_sm()
               << "\n#define PB_STATIC " << form::kStatic << "\n#define PB_SCORED " << (f.scored ? 1 : 0) << "\n#define PB_SHARED " << (f.shared ? 1 : 0)
               << "\n";
            if (f.stall != 0) os << "#define PB_TEST_STALL " << f.stall << "\n";
            return os.str();
        }

        std::atomic<int> g_test_stall{0};
        std::atomic<bool> g_test_share{false};

        // The form for `group` query heads of each key head: 16 share a tile's
        // loads, 8 where 16 would leave the ring less than three units.
        form form_of(const kv_cache& c, int64_t group) {
            form f;
            f.heads = static_cast<int>(c.heads);
            f.dim = static_cast<int>(c.dim);
            f.page = static_cast<int>(c.page_size);
            f.type = c.type;
            f.tiles8 = group > 8 ? 2 : 1;
            if (f.ring() < 3) f.tiles8 = 1;
            return f;
        }

        const char kAttention[] = "pb_paged_attention";
        const char kFinish[] = "pb_paged_finish";
        const char kSharedFinish[] = "pb_shared_finish";

        op_kernel& kernel_of(const char* name, const form& f, uint32_t smem) {
            const op_key key{reinterpret_cast<int64_t>(name), f.heads, f.dim, f.page, static_cast<int64_t>(f.type), f.scored, f.tiles8, f.join_threads, f.stall, f.shared};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = name;
                k.source = std::string{kernel_prelude()} + defines(f) + device_source();
                k.smem = smem;
            });
        }

        // Even runs of tiles (of 64 slots, but for 8 bits), over all rows one after the other, where a
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

        schedule make_schedule(const std::vector<int64_t>& lengths, int64_t heads, int64_t chunks, int64_t ctas, int64_t tile) {
            schedule r;
            const int64_t per = heads * chunks;
            int64_t total = 0, rows = 0, most = 0;
            for (int64_t length : lengths) {
                const int64_t tiles = (length + tile - 1) / tile;
                total += tiles * per;
                most = std::max(most, tiles);
                if (tiles != 0) rows += per;
            }
            const bool whole = most * tile <= kWholeRow * 64 && rows <= ctas;
            // The tile, in the order of all rows, that each CTA begins with.
            std::vector<int64_t> starts;
            if (!whole) {
                const int64_t n = std::min(total, ctas);
                int64_t row_cost = 0, row_tile = 0, cut = 0; // where the row begins
                for (int64_t length : lengths) {
                    const int64_t tiles = (length + tile - 1) / tile;
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
                const int64_t tiles = (lengths[s] + tile - 1) / tile;
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

        // Rows of `tiles` tiles each (none is empty) in even runs over at most
        // `ctas` CTAs, a row counting as `extra` tiles more than it has. Parts, a CTA's
        // run of one row each, are numbered in the CTAs' order, so that a row's
        // lie one behind the other.
        struct runs {
            std::vector<int32_t> work; // per CTA: row, tile, tiles, its first part
            std::vector<int32_t> rows; // per row: its first part, how many
            int64_t parts = 0;
        };
        constexpr int64_t kRowCost = 2; // of 128 queries: they are split, and results stored
        runs share_out(const std::vector<int64_t>& tiles, int64_t ctas, int64_t extra) {
            runs r;
            int64_t cost = 0;
            for (int64_t t : tiles) cost += t + extra;
            const int64_t n = std::min(ctas, cost - extra * static_cast<int64_t>(tiles.size()));
            r.rows.resize(2 * tiles.size(), 0);
            int64_t at = 0, cut = 1; // cost so far; the next CTA's number
            bool open = false;       // a CTA has begun
            auto begin = [&](size_t row, int64_t tile) {
                for (int64_t v : {static_cast<int64_t>(row), tile, int64_t{0}, r.parts}) r.work.push_back(static_cast<int32_t>(v));
                open = true;
            };
            for (size_t row = 0; row < tiles.size(); ++row) {
                r.rows[2 * row] = static_cast<int32_t>(r.parts);
                int64_t tile = 0;
                while (tile < tiles[row]) {
                    if (!open) begin(row, tile);
                    // Tiles up to where the next CTA begins; one at least, so that none is empty.
                    const int64_t until = cut < n ? static_cast<int64_t>(static_cast<__int128>(cost) * cut / n) - at - extra : tiles[row];
                    const int64_t take = std::min(tiles[row], std::max(until, tile + 1)) - tile;
                    r.work[r.work.size() - 2] += static_cast<int32_t>(take);
                    tile += take;
                    ++r.parts;
                    ++r.rows[2 * row + 1];
                    if (cut < n && at + extra + tile >= static_cast<int64_t>(static_cast<__int128>(cost) * cut / n)) {
                        ++cut;
                        open = false;
                    }
                }
                at += tiles[row] + extra;
            }
            return r;
        }

    } // namespace

    namespace {

        // Whether prefixes are worked through 128 queries at a time: where more
        // than 16, which the other form has, read one.
        bool prefix_stage(const kv_batch& batch, int64_t group) {
            int64_t most = 0;
            for (const auto& g : batch.groups) most = std::max(most, g.members * group);
            return prefix_attention_takes(*batch.cache) && most > 16;
        }

        // The form of what follows the prefixes, and of prefixes without a stage of
        // their own: 16 queries share a tile's loads where there are as many.
        form shared_form(const kv_batch& batch, int64_t group) {
            form f = form_of(*batch.cache, group);
            f.shared = true;
            if (prefix_stage(batch, group)) return f;
            int64_t most = group;
            for (const auto& g : batch.groups) most = std::max(most, g.members * group);
            f.tiles8 = most > 8 ? 2 : 1;
            if (f.ring() < 3) f.tiles8 = 1;
            return f;
        }

        // Whether working through the prefixes once pays, by an estimate of both sides in
        // us. Either way a row of up to 8 queries (16 where there are more) takes
        // `pass8` (`pass16`) for each MB of keys and values that it works through, most
        // of which the L2 cache delivers; sharing makes fewer rows of the prefixes, 128
        // queries each where they have a launch of their own, and takes `start` for the
        // launches and parts that it adds, and `joined` for each million channels that
        // are joined. Fitted to 398 batches of 2 to 64 sequences, inputs rotated past the
        // L2 cache; for 16 of them it takes what took over 5 % (at most 29 %) longer. 32
        // query heads over 8 of 128 channels, shared and by themselves: in bfloat16 2
        // sequences behind 16384 slots 20.0 and 24.1 us, 8 behind 2048 19.7 and 14.4,
        // behind 8192 26.9 and 39.8, 64 behind 256 20.7 and 17.7, behind 512 21.3 and
        // 26.9; in float32 64 behind 256 37.6 and 26.8, behind 1024 54.8 and 68.5; in 8
        // bits 64 behind 1024 30.1 and 28.8, behind 2048 40.5 and 46.5.
        bool worth_sharing(const kv_batch& batch, int64_t group) {
            if (batch.groups.empty()) return false;
            if (batch.always_share) return true;
            struct rates {
                double start, joined, pass8, pass16;
            };
            constexpr rates kF32{2.5, 34, 0.078, 0.135}, kBf16{4.0, 17, 0.094, 0.19}, kI8{3.9, 17, 0.070, 0.122},
                kI8Wide{7.0, 24, 0.069, 0.19}, // tiles of 64 slots
                kStage{5.0, 7.4, 0.085, 0.156};
            constexpr double kPass128 = 0.325;
            const kv_cache& c = *batch.cache;
            const bool stage = prefix_stage(batch, group);
            const rates& r = stage ? kStage
                                   : (c.type == cache_type::f32 ? kF32 : (c.type == cache_type::bf16 ? kBf16 : (tile_of(c.type, c.dim) == 128 ? kI8 : kI8Wide)));
            const form apart = form_of(c, group), together = shared_form(batch, group);
            const int64_t per = stage ? 128 : 8 * together.tiles8; // queries that read a prefix together
            const double alone = apart.tiles8 == 2 ? r.pass16 : r.pass8;
            const double shared = stage ? kPass128 : (together.tiles8 == 2 ? r.pass16 : r.pass8);
            double spared = 0; // us for each MB of a slot
            for (const auto& g : batch.groups)
                spared += static_cast<double>(g.slots) * (static_cast<double>(g.members * apart.chunks(static_cast<int>(group))) * alone -
                                                          static_cast<double>((g.members * group + per - 1) / per) * shared);
            const double slot = static_cast<double>(c.heads * 2 * c.dim * c.width()) * 1e-6;
            const double channels = static_cast<double>(batch.sequences() * c.heads * group * c.dim) * 1e-6;
            return spared * slot > r.start + r.joined * channels;
        }

        // How many CTAs (SMs) work through prefixes in their own launch, while what
        // follows them has the other SMs, `per` CTAs each, and then all. 32 query heads
        // over 8 of 128 channels, inputs rotated past the L2 cache: 64 sequences of 400
        // slots behind 16384 take 69.5 us where the prefix has all SMs but 4, 67.0
        // without a third, 79.6 without half; of 777 82, 85 and 81; of 256 behind 4096
        // 40.4, 41.5 and 37.7; of 400 behind 2048 42 each. So it goes without 4, or, if
        // there are more tiles than one for each CTA, without what looks better by this
        // estimate, in us: a tile of 128 channels takes 2.3 of a prefix and 0.78 of the
        // rest, by an SM's CTAs together, a quarter more where all SMs share HBM; CTAs
        // come and go in waves. It took the best of the three for these four.
        int64_t prefix_ctas(int64_t tiles, int64_t rows, int64_t rest, int64_t per, int64_t dim, int64_t sms) {
            const int64_t most = std::max<int64_t>(1, sms - 4), runs = per * sms;
            if (rest <= runs) return rest == 0 ? sms : most;
            const double width = static_cast<double>(dim) / 128;
            const double wave = 1 + static_cast<double>(rest) / static_cast<double>(runs) * 0.78 * static_cast<double>(per) * width;
            auto takes = [&](int64_t ctas) {
                ctas = std::min(ctas, tiles);
                const double prefix = 4 + static_cast<double>(tiles + kRowCost * rows) / static_cast<double>(ctas) * 2.3 * width;
                double t = 0;
                int64_t left = runs;
                for (int i = 1, j = 1; left > 0;) { // the next CTAs to end: of the other SMs, or after a prefix
                    const double apart = i * wave, after = prefix + j * 1.25 * wave;
                    const bool first = apart <= after;
                    left -= per * (first ? sms - ctas : ctas);
                    t = first ? apart : after;
                    ++(first ? i : j);
                }
                return std::max(t, prefix);
            };
            int64_t best = most;
            double least = 0.97 * takes(most);
            for (int64_t part : {3, 2}) {
                const int64_t ctas = std::max<int64_t>(1, sms - (sms + part - 1) / part);
                const double t = takes(ctas);
                if (t >= least) continue;
                best = ctas;
                least = t;
            }
            return best;
        }

        // The plan for `group` query heads of each key head, which the cache's next
        // such batch gets.
        const shared_plan& shared_plan_of(kv_batch& batch, int64_t group) {
            if (batch.plans->hint != nullptr) {
                std::scoped_lock lock{batch.plans->hint->mutex};
                batch.plans->hint->group = group;
            }
            std::scoped_lock lock{batch.plans->mutex};
            for (const auto& p : batch.plans->shared)
                if (p->group == group) return *p;
            const kv_cache& c = *batch.cache;
            const form f = shared_form(batch, group);
            const bool own_stage = prefix_stage(batch, group);
            auto p = std::make_unique<shared_plan>();
            p->group = group;
            p->rest.per = 8 * f.tiles8;
            p->prefix.per = own_stage ? 128 : p->rest.per;
            const int64_t heads = c.heads, n = batch.sequences();
            std::vector<int32_t> rows;
            std::vector<int64_t> tiles;
            std::vector<int32_t> outs(static_cast<size_t>(4 * n * heads), -1);
            auto put = [&](int64_t per, int64_t seq, int64_t h, int64_t begin, int64_t end, int64_t first, int64_t queries) {
                const auto row = static_cast<int32_t>(rows.size() / 8);
                for (int64_t f0 = 0; f0 < queries; f0 += per)
                    for (int64_t v : {seq, h, begin, end, first, f0, std::min(per, queries - f0), int64_t{0}})
                        rows.push_back(static_cast<int32_t>(v));
                const int64_t tile = per == 128 ? 128 : f.tile(); // slots
                if (end > begin) tiles.insert(tiles.end(), static_cast<size_t>((queries + per - 1) / per), (end - begin + tile - 1) / tile);
                return row;
            };
            std::vector<int64_t> begin(static_cast<size_t>(n), 0);
            for (const auto& g : batch.groups)
                for (int64_t h = 0; h < heads; ++h) {
                    const int32_t row = put(p->prefix.per, g.first, h, 0, g.slots, g.first, g.members * group);
                    for (int64_t s = g.first; s < g.first + g.members; ++s) {
                        begin[static_cast<size_t>(s)] = g.slots;
                        outs[static_cast<size_t>(4 * (s * heads + h) + 1)] = row;
                        outs[static_cast<size_t>(4 * (s * heads + h) + 2)] = static_cast<int32_t>((s - g.first) * group);
                    }
                }
            runs first;
            const auto prefix_rows = static_cast<int32_t>(tiles.size());
            if (own_stage) {
                int64_t rest = 0, all = 0; // tiles
                for (int64_t s = 0; s < n; ++s)
                    rest += (batch.lengths[static_cast<size_t>(s)] - begin[static_cast<size_t>(s)] + f.tile() - 1) / f.tile();
                rest *= heads * ((group + p->rest.per - 1) / p->rest.per);
                for (int64_t t : tiles) all += t;
                first = share_out(tiles, prefix_ctas(all, prefix_rows, rest, f.per_sm(), c.dim, sm_count(c.device)), kRowCost);
                tiles.clear();
            }
            for (int64_t s = 0; s < n; ++s) {
                const int64_t from = begin[static_cast<size_t>(s)], to = batch.lengths[static_cast<size_t>(s)];
                if (to > from)
                    for (int64_t h = 0; h < heads; ++h)
                        outs[static_cast<size_t>(4 * (s * heads + h))] = put(p->rest.per, s, h, from, to, s, group);
            }
            expect(rows.size() / 8 < (size_t{1} << 27), "paged_attention: too many sequences and heads");
            runs r = share_out(tiles, int64_t{f.per_sm()} * sm_count(c.device), 1);
            p->prefix.parts = first.parts;
            p->prefix.ctas = static_cast<int64_t>(first.work.size() / 4);
            p->rest.parts = r.parts;
            // Each launch counts its rows from its first.
            std::vector<int32_t> parts = first.rows;
            parts.insert(parts.end(), r.rows.begin(), r.rows.end());
            const int32_t rest_row = own_stage ? prefix_rows : 0;
            // Rows without slots, whose CTAs write zeros, come last.
            for (int64_t s = 0; s < n; ++s)
                if (batch.lengths[static_cast<size_t>(s)] == 0)
                    for (int64_t h = 0; h < heads; ++h) {
                        const int32_t row = put(p->rest.per, s, h, 0, 0, s, group);
                        for (int64_t i = 0; i < (group + p->rest.per - 1) / p->rest.per; ++i)
                            for (int32_t v : {static_cast<int32_t>(row - rest_row + i), 0, 0, 0}) r.work.push_back(v);
                    }
            p->rest.ctas = static_cast<int64_t>(r.work.size() / 4);
            for (int64_t i = 0; i < n * heads; ++i) { // the most parts of a query
                int64_t count = 0;
                for (int64_t of : {0, 1}) {
                    const int32_t row = outs[static_cast<size_t>(4 * i + of)];
                    const int64_t skip = of == 1 ? outs[static_cast<size_t>(4 * i + 2)] : 0;
                    int64_t most = 0;
                    const int64_t per = of == 1 ? p->prefix.per : p->rest.per;
                    if (row >= 0)
                        for (int64_t f = skip / per; f <= (skip + group - 1) / per; ++f)
                            most = std::max<int64_t>(most, parts[static_cast<size_t>(2 * (row + f) + 1)]);
                    count += most;
                }
                p->most_parts = std::max(p->most_parts, count);
            }
            // Rows, work and outs are read 16 bytes at a time, parts 8.
            std::vector<int32_t> host = std::move(rows);
            auto add = [&](const std::vector<int32_t>& v) {
                const size_t at = host.size();
                host.insert(host.end(), v.begin(), v.end());
                return at * 4;
            };
            // Units of the join: four queries of a prefix, or of a sequence without one.
            std::vector<int32_t> units;
            auto put_units = [&](int64_t seq, int64_t queries, bool shared) {
                for (int64_t h = 0; h < heads; ++h)
                    for (int64_t f0 = 0; f0 < queries; f0 += 4) {
                        const int32_t row = shared ? outs[static_cast<size_t>(4 * (seq * heads + h) + 1)] : -1;
                        for (int64_t v : {shared ? row + f0 / p->prefix.per : int64_t{-1}, f0, seq, h + (std::min<int64_t>(4, queries - f0) << 20)})
                            units.push_back(static_cast<int32_t>(v));
                    }
            };
            for (int64_t s = 0, g = 0; s < n;) {
                const bool shared = g < static_cast<int64_t>(batch.groups.size()) && batch.groups[static_cast<size_t>(g)].first == s;
                const int64_t members = shared ? batch.groups[static_cast<size_t>(g++)].members : 1;
                put_units(s, members * group, shared);
                s += members;
            }
            p->units = static_cast<int64_t>(units.size() / 4);
            const size_t prefix_work = add(first.work), rest_work = add(r.work), out = add(outs), unit = add(units), part = add(parts);
            auto stream = upload_stream(c.device);
            p->data = allocate(c.device, host.size() * sizeof(int32_t), stream);
            const uint64_t at = address(p->data);
            p->prefix.rows_at = at;
            p->rest.rows_at = at + static_cast<uint64_t>(rest_row) * 32;
            p->prefix.work_at = at + prefix_work;
            p->rest.work_at = at + rest_work;
            p->outs_at = at + out;
            p->units_at = at + unit;
            p->parts_at = at + part;
            check(pbrt_memcpy_h2d_async(c.device, at, host.data(), host.size() * sizeof(int32_t), stream->stream));
            check(pbrt_stream_synchronize(c.device, stream->stream));
            batch.plans->shared.push_back(std::move(p));
            return *batch.plans->shared.back();
        }

        // Attention of sequences that share prefixes; the operands are checked.
        tensor shared_attention(const op_operand& x, kv_batch& batch, float scale2, const std::shared_ptr<stream_ref>& stream) {
            kv_cache& c = *batch.cache;
            const int device = c.device;
            int group = static_cast<int>(x.shape[1] / c.heads);
            form f = shared_form(batch, group);
            f.stall = g_test_stall.load(std::memory_order_relaxed);
            const shared_plan& plan = shared_plan_of(batch, group);
            op_result out = new_result(x.shape, device, stream);
            // Workspace: the parts' results, and their maxima and sums; the prefixes' first.
            const size_t heads1 = static_cast<size_t>(plan.prefix.parts * plan.prefix.per), heads2 = static_cast<size_t>(plan.rest.parts * plan.rest.per);
            const size_t dim = static_cast<size_t>(c.dim);
            cuda_jit::device_buffer scratch = allocate(device, (heads1 * (dim + 4) + heads2 * (dim + 2)) * sizeof(float), stream);
            uint64_t partial1 = address(scratch), partial2 = partial1 + heads1 * dim * 4, ml1 = partial2 + heads2 * dim * 4, ml2 = ml1 + heads1 * 16;
            op_kernel* prefix = plan.prefix.ctas > 0 ? &prefix_attention_kernel(c, vector_width(x) == 4, f.stall) : nullptr;
            op_kernel* rest = plan.rest.ctas > 0 ? &kernel_of(kAttention, f, static_cast<uint32_t>(f.smem())) : nullptr;
            f.join_threads = plan.most_parts <= 32 ? 32 : 512;
            op_kernel& finishing = kernel_of(kSharedFinish, f, 0);
            if (prefix != nullptr) (void)prefix->on(device);
            if (rest != nullptr) (void)rest->on(device);
            (void)finishing.on(device);
            order_read(*cuda_jit::buffer_access::state(batch.data), stream);
            order_read(*cuda_jit::buffer_access::state(plan.data), stream);
            uint64_t err = 0, none = 0, queries = x.ptr;
            check(pbrt_error_word(device, &err));
            uint64_t rows1 = plan.prefix.rows_at, work1 = plan.prefix.work_at, rows2 = plan.rest.rows_at, work2 = plan.rest.work_at;
            uint64_t parts = plan.parts_at, outs = plan.outs_at;
            uint64_t scales_k = address(c.k) + static_cast<uint64_t>(c.values_bytes()), scales_v = address(c.v) + static_cast<uint64_t>(c.values_bytes());
            int width = static_cast<int>(batch.table_width), chunks = 0, longest = 0, pool_rows = static_cast<int>(c.pages * c.heads * c.page_size);
            int64_t q_seq = x.strides[0], q_head = x.strides[1];
            {
                std::scoped_lock lock{c.order};
                order_read(*cuda_jit::buffer_access::state(c.k), stream);
                order_read(*cuda_jit::buffer_access::state(c.v), stream);
                // What follows a prefix runs beside it on a stream of its own, behind
                // all that came before both; each kernel waits for that in the way of
                // its stream. (On one stream the second waits for the first: 64 sequences
                // of 400 slots behind 16384, 32 heads over 8 of 128, inputs rotated past
                // the L2 cache: 69.7 us so, 66.9 apart; of 256 behind 4096 40.7 and 37.5,
                // of 1 behind 2048 31.3 and 27.5; 2 of 1 behind 16384 20.0 and 20.4.)
                const bool apart = prefix != nullptr && rest != nullptr;
                const auto side = apart ? side_stream(device) : stream;
                if (apart) order_behind(stream, side);
                if (prefix != nullptr) {
                    void* params[] = {&c.map_k, &c.map_v, &queries, &rows1,  &batch.tables_at, &work1,     &partial1, &ml1,
                                      &width,   &group,   &q_seq,   &q_head, &pool_rows,       &scale2,    &err};
                    op_launch(*prefix, device, stream, {static_cast<uint32_t>(plan.prefix.ctas), 1, 1}, 384, params);
                }
                if (rest != nullptr) {
                    void* params[] = {&c.map_k, &c.map_v, &queries, &rows2, &batch.tables_at, &work2, &out.ptr, &partial2, &ml2, &none, &none,
                                      &width,   &group,   &chunks,  &q_seq, &q_head, &longest, &scale2, &err, &scales_k, &scales_v};
                    op_launch(*rest, device, side, {static_cast<uint32_t>(plan.rest.ctas), 1, 1}, 160, params);
                }
                if (apart) {
                    try {
                        order_behind(side, stream);
                    } catch (...) { // the workspace goes back to `stream`, which does not know of the launch
                        (void)pbrt_stream_synchronize(device, side->stream);
                        throw;
                    }
                }
            }
            // Without a stage of their own the prefixes' parts are among the others.
            if (prefix == nullptr) {
                partial1 = partial2;
                ml1 = ml2;
            }
            int per1 = plan.prefix.per, per2 = plan.rest.per, own = prefix != nullptr ? 1 : 0;
            uint64_t units = plan.units_at;
            int count = static_cast<int>(plan.units);
            void* params[] = {&outs, &parts, &partial1, &ml1, &partial2, &ml2, &out.ptr, &group, &per1, &per2, &own, &units, &count};
            const int64_t blocks = f.join_threads == 32 ? (plan.units * ((c.dim + 31) / 32) + 3) / 4 : x.shape[0] * x.shape[1];
            op_launch(finishing, device, stream, {static_cast<uint32_t>(blocks), 1, 1}, f.join_threads == 32 ? 128 : 512, params);
            return finish(std::move(out));
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
        expect(n * c.heads * ((shape[1] / c.heads + 7) / 8) < (int64_t{1} << 27), "paged_attention: too many sequences and heads");
        if (!scored && worth_sharing(batch, shape[1] / c.heads)) {
            std::vector<tensor> results;
            results.push_back(shared_attention(x, batch, scale2, stream));
            return results;
        }
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
            uint64_t scales_k = address(c.k) + static_cast<uint64_t>(c.values_bytes()), scales_v = address(c.v) + static_cast<uint64_t>(c.values_bytes());
            void* params[] = {&c.map_k, &c.map_v, &x.ptr, &batch.lengths_at, &batch.tables_at, &work,
                              &out.ptr, &partial, &ml, &logits, &norms, &width, &group, &chunks,
                              &x.strides[0], &x.strides[1], &longest32, &scale2, &err, &scales_k, &scales_v};
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
    void set_test_share_prefix(bool on) { g_test_share.store(on); }
    bool test_share_prefix() { return g_test_share.load(std::memory_order_relaxed); }

    std::pair<int, int> attention_shape(int64_t dim, cache_type type, int64_t group) {
        kv_cache c;
        c.dim = dim;
        c.type = type;
        const form f = form_of(c, group);
        return {f.per_sm(), f.shared_bytes()};
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
        schedule s = make_schedule(batch.lengths, batch.cache->heads, chunks, ctas, tile_of(batch.cache->type, batch.cache->dim));
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
        int64_t chunks = 0, ctas = 0, group = 0;
        {
            std::scoped_lock lock{batch.plans->hint->mutex};
            chunks = batch.plans->hint->chunks;
            ctas = batch.plans->hint->ctas;
            group = batch.plans->hint->group;
        }
        if (group != 0 && worth_sharing(batch, group)) {
            (void)shared_plan_of(batch, group);
            return;
        }
        if (chunks == 0) {
            chunks = 1;
            ctas = int64_t{form_of(*batch.cache, 1).per_sm()} * sm_count(batch.cache->device);
        }
        (void)plan_of(batch, chunks, ctas);
    }

    std::string attention_schedule(const std::vector<int64_t>& lengths, int64_t heads, int64_t chunks, int64_t ctas,
                                   int64_t dim, cache_type type) {
        const schedule s = make_schedule(lengths, heads, chunks, ctas, tile_of(type, dim));
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
              std::array<int, 4>{72, 2, 2, 32}, std::array<int, 4>{8, 4, 2, 32}, std::array<int, 4>{128, 1, 1, 64},
              std::array<int, 4>{80, 1, 2, 8}, std::array<int, 4>{256, 1, 2, 256}, std::array<int, 4>{16, 1, 1, 16}}) {
            form f;
            f.heads = 8;
            f.dim = dim;
            f.type = width == 1 ? cache_type::i8 : (width == 2 ? cache_type::bf16 : cache_type::f32);
            f.tiles8 = tiles8;
            f.page = page;
            f.shared = page == 32;
            f.join_threads = f.shared && width == 2 ? 32 : 128;
            f.scored = !f.shared;
            out.emplace_back("pb_paged_attention_" + std::to_string(dim) + (width == 1 ? "_i8_" : (width == 2 ? "_bf16_" : "_f32_")) + std::to_string(8 * tiles8) + (f.shared ? "_shared" : ""),
                             std::string{kernel_prelude()} + defines(f) + device_source());
        }
    }

} // namespace porch::detail
