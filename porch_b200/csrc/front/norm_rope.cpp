// RMS norm of query and key heads and their rotation by position, in one
// pass over the data, with the gradient.
//
// For a head x of D values, weight w, and the token's angles a_i:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R(a) (w n)
// where R turns the first `rot` values in pairs (i, i + rot/2), or
// (2i, 2i+1) when interleaved. With g = R(a)^T dy (the turn by -a):
//   dx = r (w g - n mean(w g n)),   dw = sum over tokens and heads of g n.
//
// Bound: HBM. The forward reads and writes each value once (8 B a value), the
// gradient reads x and dy and writes dx (12 B). A group of L lanes owns one
// head and holds it in registers (float4 loads of both partners of a pair, so
// the rotation needs no exchange between lanes); the only communication is
// the sum of squares, log2(L) shuffles. Sums are fp32.
//
// 16384 tokens x (32 + 8) heads x 128: 101 us = 6.69 TB/s forward (a copy: 6.46);
// 8192 tokens backward, with the weights' gradients: 82 us = 6.17 TB/s. Up to
// some thousand heads both are bound by their launches.
#include "operators.hpp"

#include <algorithm>
#include <sstream>
#include <stdexcept>

namespace porch::detail {

    namespace {

        const char* device_source() {
            return R"PB(
typedef long long pb_i64;
#define PB_R (2 * PB_R2)
#define PB_GPB (256 / PB_L)   // groups (heads in flight) per block
#define PB_UQ ((PB_HQ + PB_HPG - 1) / PB_HPG)
#define PB_UK ((PB_HK + PB_HPG - 1) / PB_HPG)

// Item i of a head: VEC values at A and VEC values at B.
#if !PB_INTER
#define PB_PI (PB_R2 / PB_VEC)
static __device__ __forceinline__ int pb_at_a(int i) { return i < PB_PI ? i * PB_VEC : PB_R + 2 * (i - PB_PI) * PB_VEC; }
static __device__ __forceinline__ int pb_at_b(int i) { return i < PB_PI ? PB_R2 + i * PB_VEC : PB_R + (2 * (i - PB_PI) + 1) * PB_VEC; }
#define PB_ITEMS (PB_PI + (PB_D - PB_R + 2 * PB_VEC - 1) / (2 * PB_VEC))
#else
static __device__ __forceinline__ int pb_at_a(int i) { return 2 * i * PB_VEC; }
static __device__ __forceinline__ int pb_at_b(int i) { return (2 * i + 1) * PB_VEC; }
#define PB_ITEMS ((PB_D + 2 * PB_VEC - 1) / (2 * PB_VEC))
#endif
#define PB_NI ((PB_ITEMS + PB_L - 1) / PB_L)

static __device__ __forceinline__ void pb_load(float* v, const float* p) {
#if PB_VEC == 4
    const float4 t = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
#elif PB_VEC == 2
    const float2 t = __ldg(reinterpret_cast<const float2*>(p));
    v[0] = t.x; v[1] = t.y;
#else
    v[0] = __ldg(p);
#endif
}
// A row of q, k or their gradients, which PB_WIDE says to start on a vector's
// boundary. Where rows do not, single loads fill the same registers, so the
// order of every sum, and so every result, depends on the sizes alone.
static __device__ __forceinline__ void pb_load_row(float* v, const float* p) {
#if PB_WIDE
    pb_load(v, p);
#else
#pragma unroll
    for (int e = 0; e < PB_VEC; ++e) v[e] = __ldg(p + e);
#endif
}
static __device__ __forceinline__ void pb_store(float* p, const float* v) {
#if PB_VEC == 4
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
#elif PB_VEC == 2
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
#else
    p[0] = v[0];
#endif
}

// One head's values: x[i][0] at A, x[i][1] at B; zero past D.
struct pb_head { float x[PB_NI][2][PB_VEC]; };

static __device__ __forceinline__ void pb_load_head(pb_head& h, const float* p, int lane, bool on) {
#pragma unroll
    for (int n = 0; n < PB_NI; ++n) {
        const int i = lane + n * PB_L, a = pb_at_a(i), b = pb_at_b(i);
#pragma unroll
        for (int e = 0; e < PB_VEC; ++e) h.x[n][0][e] = h.x[n][1][e] = 0.0f;
        if (on && i < PB_ITEMS) {
            pb_load_row(h.x[n][0], p + a);
            if (b < PB_D) pb_load_row(h.x[n][1], p + b);
        }
    }
}
static __device__ __forceinline__ void pb_store_head(float* p, const pb_head& h, int lane) {
#pragma unroll
    for (int n = 0; n < PB_NI; ++n) {
        const int i = lane + n * PB_L, a = pb_at_a(i), b = pb_at_b(i);
        if (i < PB_ITEMS) {
            pb_store(p + a, h.x[n][0]);
            if (b < PB_D) pb_store(p + b, h.x[n][1]);
        }
    }
}

// cos and sin of the token's position for this lane's items (1 and 0 where
// nothing turns). A position that is not a whole number of the table makes
// them NaN, and so the token's heads.
struct pb_angle { float c[PB_NI][2][PB_VEC], s[PB_NI][2][PB_VEC]; };

static __device__ __forceinline__ void pb_load_angle(pb_angle& g, const float* cs, const float* sn, float position,
                                                     pb_i64 P, int lane) {
    const bool good = position >= 0.0f && position < (float)P && position == truncf(position);
    const pb_i64 row = good ? min((pb_i64)position, P - 1) : 0;
    const float* c = cs + row * PB_R2;
    const float* s = sn + row * PB_R2;
    const float nan = __int_as_float(0x7fffffff);
#pragma unroll
    for (int n = 0; n < PB_NI; ++n) {
        const int i = lane + n * PB_L;
#pragma unroll
        for (int e = 0; e < PB_VEC; ++e) {
            g.c[n][0][e] = g.c[n][1][e] = good ? 1.0f : nan;
            g.s[n][0][e] = g.s[n][1][e] = good ? 0.0f : nan;
        }
        if (!good) continue;
#if !PB_INTER
        if (i < PB_PI) {
            pb_load(g.c[n][0], c + i * PB_VEC);
            pb_load(g.s[n][0], s + i * PB_VEC);
        }
#elif PB_VEC == 1
        if (2 * i < PB_R) { g.c[n][0][0] = __ldg(c + i); g.s[n][0][0] = __ldg(s + i); }
#else
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int at = v ? pb_at_b(i) : pb_at_a(i);
            if (at >= PB_R) continue;
#if PB_VEC == 4 // the table's rows are of an even number of values then
            const float2 x = __ldg(reinterpret_cast<const float2*>(c + at / 2)), y = __ldg(reinterpret_cast<const float2*>(s + at / 2));
            g.c[n][v][0] = x.x; g.c[n][v][2] = x.y;
            g.s[n][v][0] = y.x; g.s[n][v][2] = y.y;
#else
            g.c[n][v][0] = __ldg(c + at / 2);
            g.s[n][v][0] = __ldg(s + at / 2);
#endif
        }
#endif
    }
}

// y = R(a) x for SIGN = 1, R(a)^T x for SIGN = -1, in place.
static __device__ __forceinline__ void pb_turn(pb_head& h, const pb_angle& g, float sign, int lane) {
#pragma unroll
    for (int n = 0; n < PB_NI; ++n) {
#if !PB_INTER || PB_VEC == 1
        // Partners sit at the same place of A and B. Items that do not turn
        // have cos 1 and sin 0, but B's partner is then no part of the head.
#if !PB_INTER
        const bool turns = lane + n * PB_L < PB_PI;
#else
        const bool turns = 2 * (lane + n * PB_L) < PB_R;
#endif
#pragma unroll
        for (int e = 0; e < PB_VEC; ++e) {
            const float a = h.x[n][0][e], b = h.x[n][1][e], c = g.c[n][0][e], s = sign * g.s[n][0][e];
            h.x[n][0][e] = turns ? fmaf(a, c, -(b * s)) : a * c;
            h.x[n][1][e] = turns ? fmaf(b, c, a * s) : b * c;
        }
#else
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int i = lane + n * PB_L;
            const bool turns = (v ? pb_at_b(i) : pb_at_a(i)) < PB_R;
#pragma unroll
            for (int e = 0; e < PB_VEC; e += 2) {
                const float a = h.x[n][v][e], b = h.x[n][v][e + 1], c = g.c[n][v][e], s = sign * g.s[n][v][e];
                h.x[n][v][e] = turns ? fmaf(a, c, -(b * s)) : a * c;
                h.x[n][v][e + 1] = turns ? fmaf(b, c, a * s) : b * c;
            }
        }
#endif
    }
}

static __device__ __forceinline__ float pb_group_sum(float v) {
#pragma unroll
    for (int m = PB_L / 2; m > 0; m /= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

static __device__ __forceinline__ float pb_dot(const pb_head& a, const pb_head& b) {
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < PB_NI; ++n)
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int e = 0; e < PB_VEC; ++e) s = fmaf(a.x[n][v][e], b.x[n][v][e], s);
    return s;
}

struct pb_rows { const float* p; pb_i64 token, head; };

#ifdef PB_FORWARD
extern "C" __global__ void __launch_bounds__(256) pb_norm_rope(
    const float* q, const float* k, const float* qw, const float* kw, const float* cs, const float* sn,
    const float* pos, float* oq, float* ok, pb_i64 T, pb_i64 P, pb_i64 qt, pb_i64 qh, pb_i64 kt, pb_i64 kh, float eps) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x % PB_L;
    const pb_u64 units = (pb_u64)T * (PB_UQ + PB_UK);
    const pb_u64 want = (pb_u64)blockIdx.x * PB_GPB + threadIdx.x / PB_L;
    const bool on = want < units;
    const pb_u64 u = on ? want : units - 1;
    const pb_i64 t = u / (PB_UQ + PB_UK);
    const int j = (int)(u - (pb_u64)t * (PB_UQ + PB_UK));
    const bool is_q = j < PB_UQ;
    const int h0 = (is_q ? j : j - PB_UQ) * PB_HPG, heads = is_q ? PB_HQ : PB_HK;
    const float* src = is_q ? q + t * qt : k + t * kt;
    const pb_i64 step = is_q ? qh : kh;
    float* dst = is_q ? oq + t * PB_HQ * PB_D : ok + t * PB_HK * PB_D;
    pb_head x[PB_HPG], w;
    pb_angle g;
    const float position = __ldg(pos + t);
#pragma unroll
    for (int m = 0; m < PB_HPG; ++m) pb_load_head(x[m], src + (h0 + m) * step, lane, on && h0 + m < heads);
    pb_load_head(w, is_q ? qw : kw, lane, true);
    pb_load_angle(g, cs, sn, position, P, lane);
#pragma unroll
    for (int m = 0; m < PB_HPG; ++m) {
        const float r = rsqrtf(fmaf(pb_group_sum(pb_dot(x[m], x[m])), 1.0f / PB_D, eps));
#pragma unroll
        for (int n = 0; n < PB_NI; ++n)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < PB_VEC; ++e) x[m].x[n][v][e] = x[m].x[n][v][e] * r * w.x[n][v][e];
        pb_turn(x[m], g, 1.0f, lane);
        if (on && h0 + m < heads) pb_store_head(dst + (pb_i64)(h0 + m) * PB_D, x[m], lane);
    }
}
#endif

#ifdef PB_BACKWARD
// Query heads first, then key heads, each over the whole grid, so that one
// set of registers gathers a weight's gradient; a block adds its groups in
// order and writes one row of partial sums per weight, which
// pb_norm_rope_weights adds in order: the result depends on the sizes alone.
// Two blocks of an SM at once, at the price of a few spilled registers (half
// rotated heads of 96 side by side, 20833 tokens x 20: 105 us with one, 84.5 so;
// the worst loss, half rotated heads of 256: 76.4 and 79.7).
extern "C" __global__ void __launch_bounds__(256, PB_NI * PB_HPG <= 4 ? 2 : 1) pb_norm_rope_grad(
    const float* dyq, const float* dyk, const float* q, const float* k, const float* qw, const float* kw,
    const float* cs, const float* sn, const float* pos, float* dq, float* dk, float* partial, pb_i64 T, pb_i64 P,
    pb_i64 gqt, pb_i64 gqh, pb_i64 gkt, pb_i64 gkh, pb_i64 qt, pb_i64 qh, pb_i64 kt, pb_i64 kh, float eps) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ __align__(16) float sums[PB_GPB][PB_D]; // stored to in vectors
    const int lane = threadIdx.x % PB_L, group = threadIdx.x / PB_L;
    const int first = (threadIdx.x & ~31) / PB_L; // the warp's first group
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const int heads = which ? PB_HK : PB_HQ, per = which ? PB_UK : PB_UQ;
        const pb_u64 units = (pb_u64)T * per;
        pb_head w, dw;
        pb_load_head(w, which ? kw : qw, lane, true);
#pragma unroll
        for (int n = 0; n < PB_NI; ++n)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < PB_VEC; ++e) dw.x[n][v][e] = 0.0f;
        for (pb_u64 base = (pb_u64)blockIdx.x * PB_GPB; base + first < units; base += (pb_u64)gridDim.x * PB_GPB) {
            const bool on = base + group < units;
            const pb_u64 u = on ? base + group : units - 1;
            const pb_i64 t = u / (which ? PB_UK : PB_UQ);
            const int h0 = (int)(u - (pb_u64)t * per) * PB_HPG;
            const float* src = which ? k + t * kt : q + t * qt;
            const float* gsrc = which ? dyk + t * gkt : dyq + t * gqt;
            const pb_i64 step = which ? kh : qh, gstep = which ? gkh : gqh;
            float* dst = which ? dk + t * PB_HK * PB_D : dq + t * PB_HQ * PB_D;
            const float position = __ldg(pos + t);
            pb_head x[PB_HPG], g[PB_HPG];
            pb_angle a;
#pragma unroll
            for (int m = 0; m < PB_HPG; ++m) {
                pb_load_head(x[m], src + (h0 + m) * step, lane, on && h0 + m < heads);
                pb_load_head(g[m], gsrc + (h0 + m) * gstep, lane, on && h0 + m < heads);
            }
            pb_load_angle(a, cs, sn, position, P, lane);
#pragma unroll
            for (int m = 0; m < PB_HPG; ++m) {
                pb_turn(g[m], a, -1.0f, lane);
                const bool live = on && h0 + m < heads;
                const float r = rsqrtf(fmaf(pb_group_sum(pb_dot(x[m], x[m])), 1.0f / PB_D, eps));
                float inner = 0.0f;
#pragma unroll
                for (int n = 0; n < PB_NI; ++n)
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int e = 0; e < PB_VEC; ++e) {
                            const float norm = x[m].x[n][v][e] * r;
                            // Where nothing is loaded, x and g are 0 but a bad
                            // position's angles are NaN: such heads add nothing.
                            if (live) dw.x[n][v][e] = fmaf(g[m].x[n][v][e], norm, dw.x[n][v][e]);
                            x[m].x[n][v][e] = norm;
                            g[m].x[n][v][e] *= w.x[n][v][e];
                            inner = fmaf(g[m].x[n][v][e], norm, inner);
                        }
                inner = pb_group_sum(inner) * (1.0f / PB_D);
#pragma unroll
                for (int n = 0; n < PB_NI; ++n)
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int e = 0; e < PB_VEC; ++e)
                            x[m].x[n][v][e] = r * fmaf(-x[m].x[n][v][e], inner, g[m].x[n][v][e]);
                if (live) pb_store_head(dst + (pb_i64)(h0 + m) * PB_D, x[m], lane);
            }
        }
        if (which) asm volatile("griddepcontrol.launch_dependents;");
        pb_store_head(sums[group], dw, lane);
        __syncthreads();
        for (int c = threadIdx.x; c < PB_D; c += 256) {
            float s = 0.0f;
            for (int m = 0; m < PB_GPB; ++m) s += sums[m][c];
            partial[((pb_i64)which * gridDim.x + blockIdx.x) * PB_D + c] = s;
        }
        __syncthreads();
    }
}

// dw[which][c] = sum over `rows` rows of partial[which][row][c], 32 threads a
// column, each over every 32nd row, added in order.
extern "C" __global__ void __launch_bounds__(1024) pb_norm_rope_weights(const float* partial, float* dqw, float* dkw, int rows) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float sums[32][33];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32, c = blockIdx.x * 32 + x;
    float s = 0.0f;
    if (c < 2 * PB_D) {
        const float* p = partial + (pb_i64)(c / PB_D) * rows * PB_D + c % PB_D;
#pragma unroll 4
        for (int r = y; r < rows; r += 32) s += p[(pb_i64)r * PB_D];
    }
    sums[y][x] = s;
    __syncthreads();
    // Warp y adds column y's 32 sums.
    s = sums[x][y];
#pragma unroll
    for (int m = 16; m > 0; m /= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
    const int column = blockIdx.x * 32 + y;
    if (x == 0 && column < 2 * PB_D) (column < PB_D ? dqw : dkw)[column % PB_D] = s;
}
#endif
)PB";
        }

        struct shape_key {
            int dim = 0, half = 0, q_heads = 0, k_heads = 0, vec = 1, lanes = 1, per = 1;
            bool interleaved = false, wide = true;
        };

        int items_of(const shape_key& s) {
            if (s.interleaved) return (s.dim + 2 * s.vec - 1) / (2 * s.vec);
            return s.half / s.vec + (s.dim - 2 * s.half + 2 * s.vec - 1) / (2 * s.vec);
        }

        std::string defines(const shape_key& s) {
            std::ostringstream os;
            os << "#define PB_D " << s.dim << "\n#define PB_R2 " << s.half << "\n#define PB_HQ " << s.q_heads
               << "\n#define PB_HK " << s.k_heads << "\n#define PB_VEC " << s.vec << "\n#define PB_L " << s.lanes
               << "\n#define PB_HPG " << s.per << "\n#define PB_INTER " << (s.interleaved ? 1 : 0)
               << "\n#define PB_WIDE " << (s.wide ? 1 : 0) << "\n";
            return os.str();
        }

        std::string source_of(const shape_key& s, const char* part) {
            return std::string{kernel_prelude()} + "#define " + part + " 1\n" + defines(s) + device_source();
        }

        const char kNormRope[] = "pb_norm_rope";
        const char kNormRopeGrad[] = "pb_norm_rope_grad";
        const char kNormRopeWeights[] = "pb_norm_rope_weights";

        op_kernel& kernel_of(const shape_key& s, const char* name, const char* part) {
            const op_key key{reinterpret_cast<int64_t>(name), s.dim, s.half, s.q_heads, s.k_heads, s.vec, s.lanes,
                             s.per, s.interleaved, s.wide};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = name;
                k.source = source_of(s, part);
            });
        }

        void expect(bool ok, const char* message) {
            if (!ok) throw std::invalid_argument(message);
        }

        struct checked {
            index_t tokens = 0, table = 0;
            shape_key key;
        };

        // Every check that needs no device.
        checked check_args(const norm_rope_args& a) {
            const auto q = a.q->shape(), k = a.k->shape();
            expect(q.size() == 3 && k.size() == 3, "qk_norm_rope: q and k must be [tokens, heads, head_dim]");
            expect(q[0] == k[0] && q[2] == k[2], "qk_norm_rope: q and k must have the same tokens and head_dim");
            expect(q[1] >= 1 && k[1] >= 1 && q[1] <= 65536 && k[1] <= 65536, "qk_norm_rope: q and k need 1 to 65536 heads");
            expect(q[2] >= 1 && q[2] <= 1024, "qk_norm_rope: head_dim must be 1 to 1024");
            expect(has_shape(*a.q_weight, {q[2]}) && has_shape(*a.k_weight, {q[2]}), "qk_norm_rope: weights must be [head_dim]");
            const auto c = a.cos->shape();
            expect(c.size() == 2 && has_shape(*a.sin, {c[0], c[1]}), "qk_norm_rope: cos and sin must be [positions, rot / 2]");
            expect(c[0] >= 1 && c[1] >= 1 && 2 * c[1] <= q[2], "qk_norm_rope: rot must be 2 to head_dim, of at least one position");
            expect(c[0] <= (index_t{1} << 24), "qk_norm_rope: at most 2^24 positions (float32 counts them exactly)");
            expect(has_shape(*a.positions, {q[0]}), "qk_norm_rope: positions must be [tokens]");
            expect(a.eps >= 0.0F, "qk_norm_rope: eps must not be negative");
            checked r;
            r.tokens = q[0];
            r.table = c[0];
            r.key.dim = static_cast<int>(q[2]);
            r.key.half = static_cast<int>(c[1]);
            r.key.q_heads = static_cast<int>(q[1]);
            r.key.k_heads = static_cast<int>(k[1]);
            r.key.interleaved = a.interleaved;
            return r;
        }

        // Vectors as wide as the sizes let both partners of a pair, and the
        // table's rows, start on; lanes for one item each, up to a warp.
        // `aligned`: the width at which every row of the operands starts.
        // `few`: of 4 to 32 lanes the number that leaves the fewest idle, the
        // larger of equals. Head sizes of 80 and 96 have 10 and 12 items: 4
        // lanes of three take 60 and 54 us forward where 16 of one take 67 and
        // 61 (25000 and 20833 tokens x 20 heads, rotated whole), but 77 and 61
        // where 16 take 61 and 56 with pairs side by side, and 133 and 113 where
        // 16 take 105 and 97 in the gradient, whose registers then hold one head
        // at once.
        void choose_lanes(shape_key& s, int aligned, bool few) {
            s.vec = 4;
            while (s.vec > 1 && (s.dim % s.vec != 0 || (s.interleaved ? (2 * s.half) % s.vec : s.half % s.vec) != 0))
                s.vec /= 2;
            s.wide = aligned >= s.vec;
            const int items = items_of(s);
            s.lanes = 1;
            while (s.lanes < 32 && s.lanes < items) s.lanes *= 2;
            if (!few) return;
            for (int lanes = s.lanes / 2; lanes >= 4; lanes /= 2) {
                const int each = (items + lanes - 1) / lanes, now = (items + s.lanes - 1) / s.lanes;
                if (each <= 4 && each * lanes < now * s.lanes) s.lanes = lanes;
            }
        }

        // Heads of a token that a group takes at once, sharing its angles and
        // weights and having all their loads on the way together: as many as
        // its registers hold, once there are heads enough to fill the GPU so.
        // Forward, 16384 tokens x 40 heads of 128: 112 us with one, 98 with
        // two, 98 with four. Gradient, 8192 tokens: 84, 89 and 70 us (1021 and
        // 777 tokens: 7.0, 6.1, 6.7 and 9.1, 8.3, 9.3).
        int heads_at_once(const shape_key& s, int64_t tokens, int most, int sms) {
            const int items = (items_of(s) + s.lanes - 1) / s.lanes;
            if (tokens * (s.q_heads + s.k_heads) < int64_t{32} * sms) return 1;
            int n = most;
            while (n > 1 && n * items > most) n /= 2;
            return n;
        }

        struct operands {
            op_operand q, k, qw, kw, cos, sin, pos;
        };

        operands load(const norm_rope_args& a, const std::shared_ptr<stream_ref>& stream) {
            return {operand(*a.q, stream, true),         operand(*a.k, stream, true),
                    operand(*a.q_weight, stream, false), operand(*a.k_weight, stream, false),
                    operand(*a.cos, stream, false),      operand(*a.sin, stream, false),
                    operand(*a.positions, stream, false)};
        }

    } // namespace

    std::array<tensor, 2> qk_norm_rope(const norm_rope_args& a) {
        checked c = check_args(a);
        const int device = device_of(*a.q, "qk_norm_rope");
        auto stream = current_stream(device);
        operands x = load(a, stream);
        op_result oq = new_result(x.q.shape, device, stream), ok = new_result(x.k.shape, device, stream);
        if (c.tokens != 0) {
            shape_key& s = c.key;
            choose_lanes(s, std::min(vector_width(x.q), vector_width(x.k)), !a.interleaved);
            s.per = heads_at_once(s, c.tokens, 2, sm_count(device));
            op_kernel& kernel = kernel_of(s, kNormRope, "PB_FORWARD");
            const int64_t units = c.tokens * ((s.q_heads + s.per - 1) / s.per + (s.k_heads + s.per - 1) / s.per);
            const int64_t blocks = (units + 256 / s.lanes - 1) / (256 / s.lanes);
            expect(blocks <= 0x7fffffff, "qk_norm_rope: too many tokens");
            float eps = a.eps;
            void* params[] = {&x.q.ptr,       &x.k.ptr,         &x.qw.ptr,        &x.kw.ptr,
                              &x.cos.ptr,     &x.sin.ptr,       &x.pos.ptr,       &oq.ptr,
                              &ok.ptr,        &c.tokens,        &c.table,         &x.q.strides[0],
                              &x.q.strides[1], &x.k.strides[0], &x.k.strides[1],  &eps};
            op_launch(kernel, device, stream, {static_cast<uint32_t>(blocks), 1, 1}, 256, params);
        }
        return {finish(std::move(oq)), finish(std::move(ok))};
    }

    std::array<tensor, 4> qk_norm_rope_backward(const tensor& dq, const tensor& dk, const norm_rope_args& a) {
        checked c = check_args(a);
        expect(std::ranges::equal(dq.shape(), a.q->shape()) && std::ranges::equal(dk.shape(), a.k->shape()),
               "qk_norm_rope_backward: gradients must have the shapes of q and k");
        const int device = device_of(*a.q, "qk_norm_rope_backward");
        auto stream = current_stream(device);
        operands x = load(a, stream);
        op_operand gq = operand(dq, stream, true), gk = operand(dk, stream, true);
        op_result oq = new_result(x.q.shape, device, stream), ok = new_result(x.k.shape, device, stream);
        op_result wq = new_result({c.key.dim}, device, stream), wk = new_result({c.key.dim}, device, stream);
        if (c.tokens == 0) {
            check(pbrt_memset_d32_async(device, wq.ptr, 0, static_cast<size_t>(c.key.dim), stream->stream));
            check(pbrt_memset_d32_async(device, wk.ptr, 0, static_cast<size_t>(c.key.dim), stream->stream));
        } else {
            shape_key& s = c.key;
            choose_lanes(s, std::min({vector_width(x.q), vector_width(x.k), vector_width(gq), vector_width(gk)}), false);
            s.per = heads_at_once(s, c.tokens, 4, sm_count(device));
            op_kernel& kernel = kernel_of(s, kNormRopeGrad, "PB_BACKWARD");
            op_kernel& weights = kernel_of(s, kNormRopeWeights, "PB_BACKWARD");
            const int64_t groups = 256 / s.lanes;
            const int64_t units = c.tokens * ((std::max(s.q_heads, s.k_heads) + s.per - 1) / s.per);
            // Two blocks of an SM: fewer partial sums to add (of three to
            // eight, none was faster).
            const int64_t blocks = std::min<int64_t>((units + groups - 1) / groups, int64_t{2} * sm_count(device));
            auto partial = allocate(device, static_cast<size_t>(2 * blocks * s.dim) * sizeof(float), stream);
            uint64_t pp = address(partial);
            float eps = a.eps;
            int rows = static_cast<int>(blocks);
            void* params[] = {&gq.ptr,          &gk.ptr,          &x.q.ptr,         &x.k.ptr,         &x.qw.ptr,
                              &x.kw.ptr,        &x.cos.ptr,       &x.sin.ptr,       &x.pos.ptr,       &oq.ptr,
                              &ok.ptr,          &pp,              &c.tokens,        &c.table,         &gq.strides[0],
                              &gq.strides[1],   &gk.strides[0],   &gk.strides[1],   &x.q.strides[0],  &x.q.strides[1],
                              &x.k.strides[0],  &x.k.strides[1],  &eps};
            op_launch(kernel, device, stream, {static_cast<uint32_t>(blocks), 1, 1}, 256, params);
            void* wparams[] = {&pp, &wq.ptr, &wk.ptr, &rows};
            op_launch(weights, device, stream, {static_cast<uint32_t>((2 * s.dim + 31) / 32), 1, 1}, 1024, wparams);
        }
        return {finish(std::move(oq)), finish(std::move(ok)), finish(std::move(wq)), finish(std::move(wk))};
    }

    void norm_rope_sources(std::vector<std::pair<std::string, std::string>>& out) {
        for (const auto& [dim, rot, inter, aligned] :
             {std::array<int, 4>{128, 128, 0, 4}, std::array<int, 4>{80, 40, 1, 1}, std::array<int, 4>{37, 18, 0, 1},
              std::array<int, 4>{37, 18, 1, 1},
              std::array<int, 4>{1023, 1022, 0, 4}, std::array<int, 4>{96, 48, 0, 4}, std::array<int, 4>{512, 64, 0, 4}}) {
            shape_key s;
            s.dim = dim;
            s.half = rot / 2;
            s.q_heads = 5;
            s.k_heads = 2;
            s.interleaved = inter != 0;
            choose_lanes(s, aligned, inter == 0);
            s.per = heads_at_once(s, 1 << 20, aligned, 148);
            const std::string tag = "_" + std::to_string(dim) + (inter ? "i" : "h");
            out.emplace_back("pb_norm_rope" + tag, source_of(s, "PB_FORWARD"));
            out.emplace_back("pb_norm_rope_grad" + tag, source_of(s, "PB_BACKWARD"));
        }
    }

} // namespace porch::detail
