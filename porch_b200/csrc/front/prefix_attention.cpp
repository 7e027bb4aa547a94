// Attention of many queries over one run of slots that they all see: the shared
// prefix of a batch, for a bfloat16 cache, on the tensor cores' large tiles.
//
// A row is one key head of a prefix with up to 128 of the queries that read it
// (several sequences' heads); for each 128 slots
//   S = Q K^T,  P = 2^(S - m),  O = O 2^(m' - m) + P V
// with m the running maximum of each query and S in units of log2 (the scale is
// part of Q). Queries and weights are three bfloat16 terms each, their upper,
// middle and lower 8 bits, so that products with the cache's values are exact;
// smaller terms are added first. The accumulators cut low bits, so those of a
// tile start from zero and are added to the running sums in fp32, rounded to
// nearest.
//
// One CTA an SM, 384 threads:
//   warp 0      loads K and V of each tile through a ring of TMA units, in the
//               order in which they are used: K0 K1 V0 K2 V1 ...; slots past the
//               run's end are filled with zeros;
//   warp 1      allocates tensor memory and issues the MMAs, S a tile ahead;
//   warps 4-11  two threads for each query: they read S, add the O of the tile
//               before to the running sums in their registers, and put P's terms
//               to tensor memory, where P V takes them from; they split a row's
//               queries.
// So tensor cores run P V while the exponentials of the next tile are formed, and
// the S after that while O is read and P written. Tensor memory: S 128 columns, P
// 3 x 64, O 128.
//
// Bound: tensor cores and the shared memory that feeds them. With three terms S and
// P V are 6 products of 128 x 128 x head_dim a tile where the formula has 2. 64
// sequences behind 16384 slots, 32 heads of 128 over 8: 43 to 46 us on every SM with
// the tensor pipe 68 % busy (it leaves some to what follows: prefix_ctas()); a tile takes 4300 cycles, some 2100 of them S, whose operands both
// come from shared memory, and 1750 P V, whose weights come from tensor memory. Every mbarrier wait
// is bounded, and nobody leaves while loads or MMAs are in flight.
#include "operators.hpp"

#include <sstream>

namespace porch::detail {

    namespace {

        const char* device_source() {
            return R"PB(
typedef long long pb_i64;
#define PB_WAIT_CYCLES 4000000000ll
#define PB_PLANES ((PB_D + 63) / 64)
#define PB_UNIT (PB_PLANES * 16384)       // 128 slots of K or V, one 128-byte plane after the other
#define PB_QTERM (PB_PLANES * 16384)      // 128 queries, one term
#define PB_BOX (PB_PS < 64 ? PB_PS : 64)
#define PB_KSTEPS ((PB_D + 15) / 16)
#define PB_N (PB_KSTEPS * 16)             // channels of O
#define PB_NH ((PB_KSTEPS + 1) / 2 * 16)  // of them, the first half's
#define PB_S 0                            // tensor memory columns
#define PB_P(term) (128 + (term) * 64)
#define PB_O 320
#define PB_LOWEST __int_as_float(0xff7fffff)

// Of the launch's 168 registers a thread, 128 threads keep 56, and 256 get 224.
#define PB_REGISTERS_LESS asm volatile("setmaxnreg.dec.sync.aligned.u32 56;")
#define PB_REGISTERS_MORE asm volatile("setmaxnreg.inc.sync.aligned.u32 224;")

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
// Bounded wait: false when the budget ran out or another role gave up.
static __device__ __forceinline__ bool pb_wait(pb_u32 bar, pb_u32 parity, volatile int* abort_flag, int* err, int site) {
    if (pb_mbar_try(bar, parity)) return true;
    const long long start = clock64();
    for (;;) {
        if (pb_mbar_try(bar, parity)) return true;
        if (*abort_flag) return false;
        if (clock64() - start > PB_WAIT_CYCLES) {
            *abort_flag = 1;
            if (atomicCAS(err, 0, 0x7d40 + site) == 0) {
                err[1] = site;
                err[2] = (int)blockIdx.x;
            }
            return false;
        }
    }
}
// Teardown wait: bounded, records nothing.
static __device__ __forceinline__ void pb_wait_quiet(pb_u32 bar, pb_u32 parity) {
    const long long start = clock64();
    while (!pb_mbar_try(bar, parity) && clock64() - start <= PB_WAIT_CYCLES) {
    }
}
static __device__ __forceinline__ void pb_tma_load(pb_u32 dst, const pb_tmap* map, pb_u32 bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 :: "r"(dst), "l"((unsigned long long)map), "r"(bar), "r"(x), "r"(y) : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle, 8-row groups 1024 bytes
// apart. K-major (queries, keys): a k-step of 16 channels is 32 bytes further in
// the swizzled row. Values are contiguous along their channels (N): 64 of them a
// plane, the planes 16384 bytes apart, and a k-step is 16 rows, 2048 bytes.
static __device__ __forceinline__ pb_u64 pb_desc(pb_u32 addr, pb_u32 leading) {
    return (pb_u64)((addr & 0x3FFFFu) >> 4) | (pb_u64)(leading >> 4) << 16 | (pb_u64)(1024 >> 4) << 32 | (pb_u64)1 << 46 |
           (pb_u64)2 << 61;
}
// Instruction descriptors: D f32, A and B bf16, M = 128; B of P V is N-major.
#define PB_IDESC_S ((1u << 4) | (1u << 7) | (1u << 10) | ((pb_u32)(128 >> 3) << 17) | ((pb_u32)(128 >> 4) << 24))
#define PB_IDESC_O ((1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((pb_u32)(PB_N >> 3) << 17) | ((pb_u32)(128 >> 4) << 24))
static __device__ __forceinline__ void pb_mma_shared(pb_u32 d, pb_u64 a, pb_u64 b, pb_u32 accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 :: "r"(d), "l"(a), "l"(b), "r"(PB_IDESC_S), "r"(accumulate) : "memory");
}
static __device__ __forceinline__ void pb_mma_tensor(pb_u32 d, pb_u32 a, pb_u64 b, pb_u32 accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 :: "r"(d), "r"(a), "l"(b), "r"(PB_IDESC_O), "r"(accumulate) : "memory");
}
// Arrives on `bar` once the MMAs issued so far have completed.
static __device__ __forceinline__ void pb_commit(pb_u32 bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
// One lane of a warp that runs along whole.
static __device__ __forceinline__ bool pb_elected() {
    pb_u32 r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
static __device__ __forceinline__ float pb_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
#define PB_LD32(taddr, v)                                                                                     \
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15," \
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                   \
                 : "=f"((v)[0]), "=f"((v)[1]), "=f"((v)[2]), "=f"((v)[3]), "=f"((v)[4]), "=f"((v)[5]), "=f"((v)[6]), \
                   "=f"((v)[7]), "=f"((v)[8]), "=f"((v)[9]), "=f"((v)[10]), "=f"((v)[11]), "=f"((v)[12]), "=f"((v)[13]), \
                   "=f"((v)[14]), "=f"((v)[15]), "=f"((v)[16]), "=f"((v)[17]), "=f"((v)[18]), "=f"((v)[19]), "=f"((v)[20]), \
                   "=f"((v)[21]), "=f"((v)[22]), "=f"((v)[23]), "=f"((v)[24]), "=f"((v)[25]), "=f"((v)[26]), "=f"((v)[27]), \
                   "=f"((v)[28]), "=f"((v)[29]), "=f"((v)[30]), "=f"((v)[31])                                 \
                 : "r"(taddr))
#define PB_LD16(taddr, v)                                                                                     \
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" \
                 : "=f"((v)[0]), "=f"((v)[1]), "=f"((v)[2]), "=f"((v)[3]), "=f"((v)[4]), "=f"((v)[5]), "=f"((v)[6]), \
                   "=f"((v)[7]), "=f"((v)[8]), "=f"((v)[9]), "=f"((v)[10]), "=f"((v)[11]), "=f"((v)[12]), "=f"((v)[13]), \
                   "=f"((v)[14]), "=f"((v)[15])                                                               \
                 : "r"(taddr))
#define PB_ST16(taddr, v)                                                                                     \
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" \
                 :: "r"(taddr), "r"((v)[0]), "r"((v)[1]), "r"((v)[2]), "r"((v)[3]), "r"((v)[4]), "r"((v)[5]), "r"((v)[6]), \
                    "r"((v)[7]), "r"((v)[8]), "r"((v)[9]), "r"((v)[10]), "r"((v)[11]), "r"((v)[12]), "r"((v)[13]), \
                    "r"((v)[14]), "r"((v)[15]) : "memory")

// The next term of two values: their upper 16 bits, side by side; what is left
// of them stays, exactly (x - term in one instruction that takes the term as
// bfloat16; by masking the float first a tile's terms took half as long again).
// Cutting keeps every bit: three terms of 8 hold a float32's 24.
static __device__ __forceinline__ pb_u32 pb_term(float& a, float& b) {
    const pb_u32 w = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    asm("{\n .reg .b16 l, h, m;\n mov.b32 {l, h}, %2;\n mov.b16 m, 0xbf80;\n fma.rn.f32.bf16 %0, l, m, %0;\n"
        " fma.rn.f32.bf16 %1, h, m, %1;\n}\n" : "+f"(a), "+f"(b) : "r"(w));
    return w;
}

// A row: a run of slots of one key head, and its queries (as in pb_paged_attention).
struct pb_at { int s, h, begin, end, first, f0, count, tiles; };
static __device__ __forceinline__ pb_at pb_row(const int4* rows, int row) {
    const int4 x = rows[2 * row], y = rows[2 * row + 1];
    return {x.x, x.y, x.z, x.w, y.x, y.y, y.z, (x.w - x.z + 127) >> 7};
}

extern "C" __global__ void __launch_bounds__(384, 1) pb_prefix_attention(
    const __grid_constant__ pb_tmap map_k, const __grid_constant__ pb_tmap map_v, const float* q, const int4* rows,
    const int* tables, const int4* work, float* partial, float2* partial_ml, int width, int group, pb_i64 q_seq,
    pb_i64 q_head, int pool_rows, float scale2, int* err) {
    extern __shared__ char raw[];
    __shared__ pb_u64 bars[2 * PB_RING + 6];
    __shared__ pb_u32 tmem_slot;
    __shared__ int abort_flag;
    const pb_u32 ring = (pb_smem(raw) + 1023u) & ~1023u, queries = ring + PB_RING * PB_UNIT;
    const pb_u32 full = pb_smem(bars), empty = full + 8 * PB_RING, s_full = empty + 8 * PB_RING, s_free = s_full + 8,
                 p_ready = s_free + 8, o_full = p_ready + 8, q_ready = o_full + 8, done = q_ready + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < PB_RING; ++i) {
            pb_mbar_init(full + 8 * i, 1);
            pb_mbar_init(empty + 8 * i, 1);
        }
        pb_mbar_init(s_full, 1);
        pb_mbar_init(s_free, 256);
        pb_mbar_init(p_ready, 256);
        pb_mbar_init(o_full, 1);
        pb_mbar_init(q_ready, 256);
        pb_mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(pb_smem(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const pb_u32 tmem = tmem_slot;
    // The plan, rows and tables were in place before the launch.
    const int4 mine = work[blockIdx.x];

    if (warp < 4) PB_REGISTERS_LESS;
    if (warp == 0) {
        // ---- producer
        asm volatile("griddepcontrol.wait;" ::: "memory");
        // Every CTA has its SM by the time that all are here; the join, which is next on
        // this stream, may come in as SMs come free and waits there.
        asm volatile("griddepcontrol.launch_dependents;");
        int unit = 0, row = mine.x, tile = mine.y, left = mine.z;
        bool good = true;
        auto load = [&](const pb_tmap* map, int y) {
            const int slot = unit % PB_RING;
            good = pb_wait(empty + 8 * slot, ((unit / PB_RING) & 1) ^ 1, &abort_flag, err, 1);
            good = __all_sync(0xffffffffu, good);
            if (!good) return;
            if (lane == 0) pb_mbar_expect_tx(full + 8 * slot, PB_UNIT);
            __syncwarp();
            if (lane * PB_BOX < 128) {
#pragma unroll
                for (int c = 0; c < PB_PLANES; ++c)
                    pb_tma_load(ring + slot * PB_UNIT + c * 16384 + lane * PB_BOX * 128, map, full + 8 * slot, c * 64, y);
            }
            ++unit;
        };
        while (left > 0 && good) {
            const pb_at a = pb_row(rows, row);
            const int n = min(left, a.tiles - tile);
            int before = 0; // where the last tile's rows lie
            for (int i = 0; i <= n && good; ++i) {
                int y = pool_rows; // past the pool: zeros
                if (i < n) {
                    const int first = a.begin + (tile + i) * 128 + lane * PB_BOX;
                    if (lane * PB_BOX < 128 && first < a.end)
                        y = (tables[(pb_i64)a.s * width + first / PB_PS] * PB_H + a.h) * PB_PS + first % PB_PS;
                    load(&map_k, y);
                }
                if (i > 0 && good) load(&map_v, before);
                before = y;
            }
            left -= n;
            tile = 0;
            ++row;
        }
        // Nothing may land after this CTA is gone.
        if (lane == 0)
            for (int u = unit > PB_RING ? unit - PB_RING : 0; u < unit; ++u) pb_wait_quiet(full + 8 * (u % PB_RING), (u / PB_RING) & 1);
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMAs. In this order: S of tile t + 1, which keeps the tensor cores busy
        // while O of tile t - 1 is read and P of tile t is written, then P V of tile t
        // (by two warps they took turns at each other's, and both came late: 79 us of
        // stream for 64 sequences behind 16384 slots, 78 so). The whole warp runs
        // along, so that descriptors are known to be the same in it and stay in
        // uniform registers.
        const bool leader = pb_elected();
        const pb_u64 q_desc = pb_desc(queries, 16), k_desc = pb_desc(ring, 16), v_desc = pb_desc(ring, 16384);
        int unit = 0, row = mine.x, tile = mine.y, left = __shfl_sync(0xffffffffu, mine.z, 0), t = 0, segment = 0;
        bool good = true;
        auto take = [&]() { // the next unit's slot, once it has landed
            const int slot = __shfl_sync(0xffffffffu, unit % PB_RING, 0);
            good = good && pb_wait(full + 8 * slot, (unit / PB_RING) & 1, &abort_flag, err, 2);
            good = __all_sync(0xffffffffu, good);
            ++unit;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return slot;
        };
        auto scores = [&]() {
            const int slot = take();
            if (!good) return;
            const pb_u64 keys = k_desc + (pb_u64)(slot * (PB_UNIT >> 4));
            if (leader) {
#pragma unroll
                for (int term = 2; term >= 0; --term)
#pragma unroll
                    for (int k = 0; k < PB_KSTEPS; ++k)
                        pb_mma_shared(tmem + PB_S, q_desc + (pb_u64)((term * PB_QTERM + (k >> 2) * 16384 + (k & 3) * 32) >> 4),
                                      keys + (pb_u64)(((k >> 2) * 16384 + (k & 3) * 32) >> 4), term != 2 || k != 0);
                pb_commit(empty + 8 * slot);
                pb_commit(s_full);
            }
            __syncwarp();
        };
#if PB_TEST_STALL == 1
        if (blockIdx.x == 0) left = 0; // nothing is multiplied: the others' waits run out
#endif
        while (left > 0 && good) {
            const pb_at a = pb_row(rows, row);
            const int n = __shfl_sync(0xffffffffu, min(left, a.tiles - tile), 0);
            good = pb_wait(q_ready, segment & 1, &abort_flag, err, 3);
            scores();
            for (int i = 0; i < n && good; ++i, ++t) {
                if (i + 1 < n) {
                    good = pb_wait(s_free, t & 1, &abort_flag, err, 11);
                    scores();
                    if (!good) break;
                }
                // P is there, and the tile's before O was read.
                good = pb_wait(p_ready, t & 1, &abort_flag, err, 4);
                const int slot = take();
                if (!good) break;
                const pb_u64 values = v_desc + (pb_u64)(slot * (PB_UNIT >> 4));
                if (leader) {
#pragma unroll
                    for (int term = 2; term >= 0; --term)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            pb_mma_tensor(tmem + PB_O, tmem + PB_P(term) + k * 8, values + (pb_u64)(k * 2048 >> 4), term != 2 || k != 0);
                    pb_commit(empty + 8 * slot);
                    pb_commit(o_full);
                }
                __syncwarp();
            }
            left -= n;
            tile = 0;
            ++row;
            ++segment;
        }
        if (leader) pb_commit(done); // whether or not the loops finished
        __syncwarp();
    } else if (warp >= 4) {
        // ---- softmax and running sums: two threads for each query, of 64 slots and
        // half its channels each. Both look at all logits for the maximum, which costs
        // less than handing it over.
        PB_REGISTERS_MORE;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int query = (warp & 3) * 32 + lane, half = (warp - 4) >> 2;
        const int first = half * PB_NH; // its channels
        const pb_u32 lanes = tmem + ((pb_u32)(warp & 3) << 21);
        int row = mine.x, tile = mine.y, left = mine.z, t = 0, part = mine.w;
        bool good = true;
        while (left > 0 && good) {
            const pb_at a = pb_row(rows, row);
            const int n = min(left, a.tiles - tile);
            // The row's queries, 4 channels at a time, in units of log2; zeros past
            // the head size and the row's queries. MMAs of the row before have
            // completed: its last O was waited for. Every load before the first use.
            {
                constexpr int pieces = 128 * PB_PLANES * 16 / 256; // of a thread, every 8th or 16th row
                float4 x[pieces];
                const int r0 = (threadIdx.x - 128) / (PB_PLANES * 16), c = (threadIdx.x - 128) % (PB_PLANES * 16) * 4;
                int member = (a.f0 + r0) / group, head = (a.f0 + r0) % group;
                const int members = 16 / PB_PLANES / group, heads = 16 / PB_PLANES % group;
#pragma unroll
                for (int u = 0; u < pieces; ++u) {
                    const int r = r0 + u * (16 / PB_PLANES);
                    const float* src = q + (a.first + member) * q_seq + (a.h * group + head) * q_head + c;
                    x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (r < a.count && c < PB_D) // head sizes are whole pieces
#if PB_WIDE
                        x[u] = pb_ld4(src);
#else
                        x[u] = make_float4(__ldg(src), __ldg(src + 1), __ldg(src + 2), __ldg(src + 3));
#endif
                    member += members;
                    head += heads;
                    if (head >= group) {
                        head -= group;
                        ++member;
                    }
                }
#pragma unroll
                for (int u = 0; u < pieces; ++u) {
                    const int r = r0 + u * (16 / PB_PLANES);
                    x[u].x *= scale2;
                    x[u].y *= scale2;
                    x[u].z *= scale2;
                    x[u].w *= scale2;
                    const pb_u32 to = queries + (c >> 6) * 16384 + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4) + (c & 4) * 2;
#pragma unroll
                    for (int term = 0; term < 3; ++term) {
                        const pb_u32 low = pb_term(x[u].x, x[u].y), high = pb_term(x[u].z, x[u].w);
                        asm volatile("st.shared.v2.b32 [%0], {%1,%2};" :: "r"(to + term * PB_QTERM), "r"(low), "r"(high) : "memory");
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            pb_mbar_arrive(q_ready);
            float o[PB_NH], m = PB_LOWEST, l = 0.0f, corr = 0.0f;
#pragma unroll
            for (int j = 0; j < PB_NH; ++j) o[j] = 0.0f;
            // Adds tile u's O, whose weights were relative to the maximum after it.
            auto drain = [&](int u, float c) {
                good = __all_sync(0xffffffffu, pb_wait(o_full, u & 1, &abort_flag, err, 8));
                if (!good) return;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int k = 0; k < PB_NH; k += 16) {
                    float d[16];
                    if (first + k < PB_N) PB_LD16(lanes + PB_O + first + k, d);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (first + k < PB_N) o[k + j] = fmaf(o[k + j], c, d[j]);
                }
            };
            for (int i = 0; i < n; ++i, ++t) {
                good = __all_sync(0xffffffffu, pb_wait(s_full, t & 1, &abort_flag, err, 6));
                if (!good) break;
#if PB_TEST_STALL == 2
                if (blockIdx.x == 0) { // gives up at once, with loads and MMAs on their way
                    abort_flag = 1;
                    if (atomicCAS(err, 0, 0x7d40 + 10) == 0) err[1] = 10;
                    good = false;
                    break;
                }
#endif
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int valid = a.end - a.begin - (tile + i) * 128;
                float v[64], top[4];
                {
                    float y[64];
                    PB_LD32(lanes + PB_S + 64 * half, v);
                    PB_LD32(lanes + PB_S + 64 * half + 32, v + 32);
                    PB_LD32(lanes + PB_S + 64 * (half ^ 1), y);
                    PB_LD32(lanes + PB_S + 64 * (half ^ 1) + 32, y + 32);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (valid < 128) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) {
                            if (j + 64 * half >= valid) v[j] = __int_as_float(0xff800000);
                            if (j + 64 * (half ^ 1) >= valid) y[j] = __int_as_float(0xff800000);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) top[j] = fmaxf(v[j], y[j]);
#pragma unroll
                    for (int j = 4; j < 64; ++j) top[j & 3] = fmaxf(fmaxf(top[j & 3], v[j]), y[j]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                pb_mbar_arrive(s_free);
                const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                const float before = corr;
                corr = pb_exp2(m - now);
                m = now;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    v[j] = pb_exp2(v[j] - now);
                    sum[j & 3] += v[j];
                }
                l = fmaf(l, corr, (sum[0] + sum[1]) + (sum[2] + sum[3]));
                // The tile before: its O, after which P's place is free.
                if (i > 0) drain(t - 1, before);
                if (!good) break;
#pragma unroll
                for (int term = 0; term < 3; ++term)
#pragma unroll
                    for (int c = 0; c < 32; c += 16) {
                        pb_u32 w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = pb_term(v[2 * (c + j)], v[2 * (c + j) + 1]);
                        PB_ST16(lanes + PB_P(term) + 32 * half + c, w);
                    }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                pb_mbar_arrive(p_ready);
            }
            if (good) drain(t - 1, corr);
            if (good && query < a.count) {
                partial_ml[((pb_i64)part * 2 + half) * 128 + query] = make_float2(m, l);
                // Four channels of four queries side by side, as the join reads them: a
                // warp's stores fill whole sectors (query after query they took 4500
                // cycles of a row's end).
                float4* to = reinterpret_cast<float4*>(partial) +
                             (((pb_i64)part * 32 + (query >> 2)) * (PB_D / 4) + first / 4) * 4 + (query & 3);
#pragma unroll
                for (int j = 0; j < PB_NH; j += 4)
                    if (first + j < PB_D) to[j] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            }
            left -= n;
            tile = 0;
            ++row;
            ++part;
        }
    }
    // Every MMA issued has completed before tensor and shared memory go.
    if (threadIdx.x == 0) pb_wait_quiet(done, 0);
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
}
)PB";
        }

        int planes_of(int64_t dim) { return static_cast<int>((dim + 63) / 64); }
        int ring_of(int64_t dim) { return dim > 64 ? 4 : 8; }

        std::string source_of(const kv_cache& c, bool wide, int stall) {
            std::ostringstream os;
            os << kernel_prelude() << "#define PB_H " << c.heads << "\n#define PB_D " << c.dim << "\n#define PB_PS " << c.page_size
               << "\n#define PB_RING " << ring_of(c.dim) << "\n#define PB_WIDE " << (wide ? 1 : 0) << "\n#define PB_TEST_STALL " << stall << "\n" << device_source();
            return os.str();
        }

        const char kPrefix[] = "pb_prefix_attention";

    } // namespace

    bool prefix_attention_takes(const kv_cache& c) { return c.type == cache_type::bf16 && c.dim <= 128; }

    op_kernel& prefix_attention_kernel(const kv_cache& c, bool wide, int stall) {
        const op_key key{reinterpret_cast<int64_t>(kPrefix), c.heads, c.dim, c.page_size, wide, stall};
        return op_kernel_for(key, [&](op_kernel& k) {
            k.name = kPrefix;
            k.source = source_of(c, wide, stall);
            k.smem = static_cast<uint32_t>(1024 + planes_of(c.dim) * (ring_of(c.dim) + 3) * 16384);
        });
    }

    void prefix_attention_sources(kernel_list& out) {
        kv_cache c;
        c.heads = 8;
        c.type = cache_type::bf16;
        for (const auto& [dim, page] : {std::pair{128, 64}, std::pair{80, 8}, std::pair{64, 256}, std::pair{8, 16}}) {
            c.dim = dim;
            c.page_size = page;
            out.emplace_back("pb_prefix_attention_" + std::to_string(dim), source_of(c, dim != 80, 0));
        }
    }

} // namespace porch::detail
