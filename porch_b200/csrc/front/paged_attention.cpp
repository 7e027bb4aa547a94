// Attention of one new token per sequence over a paged cache:
//   o = softmax(scale q K^T) V
// over the slots in use, query heads sharing key heads in groups, and its
// scored form, which adds each slot's attention weight, summed over the query
// heads of its key head, to running scores (what eviction ranks slots by).
// A sequence without slots gives zeros.
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

        const char* device_source() {
            return R"PB(
typedef long long pb_i64;
#if PB_BF16
typedef unsigned short pb_cell;
static __device__ __forceinline__ float pb_value(pb_cell c) { return __uint_as_float((pb_u32)c << 16); }
#else
typedef float pb_cell;
static __device__ __forceinline__ float pb_value(pb_cell c) { return c; }
#endif

static __device__ __forceinline__ float pb_block_reduce(float v, bool maximum, float* sh) {
#pragma unroll
    for (int m = 16; m > 0; m /= 2) {
        const float o = __shfl_xor_sync(0xffffffffu, v, m);
        v = maximum ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int i = 1; i < 8; ++i) v = maximum ? fmaxf(v, sh[i]) : v + sh[i];
    return v;
}

// One block per sequence and query head: logits to `weights`, then their
// softmax in place, then the weighted sum of V.
extern "C" __global__ void __launch_bounds__(256) pb_attend(
    const float* q, const pb_cell* pk, const pb_cell* pv, const int* lengths, const int* tables, float* weights,
    float* out, pb_i64 longest, int width, int heads, int group, float scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float sh[8];
    const pb_i64 row = blockIdx.x;
    const int s = (int)(row / heads), kvh = (int)(row % heads) / group, n = lengths[s];
    const int* table = tables + (pb_i64)s * width;
    float* w = weights + row * longest;
    const float* x = q + row * PB_D;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float top = __int_as_float(0xff800000);
    for (int i = warp; i < n; i += 8) {
        const pb_cell* k = pk + (((pb_i64)table[i / PB_PS] * PB_H + kvh) * PB_PS + i % PB_PS) * PB_D;
        float a = 0.0f;
        for (int d = lane; d < PB_D; d += 32) a = fmaf(x[d], pb_value(k[d]), a);
#pragma unroll
        for (int m = 16; m > 0; m /= 2) a += __shfl_xor_sync(0xffffffffu, a, m);
        a *= scale;
        if (lane == 0) w[i] = a;
        top = fmaxf(top, a);
    }
    top = pb_block_reduce(top, true, sh);
    float sum = 0.0f;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float p = expf(w[i] - top);
        w[i] = p;
        sum += p;
    }
    sum = pb_block_reduce(sum, false, sh);
    for (int i = threadIdx.x; i < n; i += 256) w[i] /= sum;
    __syncthreads();
    for (int d = threadIdx.x; d < PB_D; d += 256) {
        float a = 0.0f;
        for (int i = 0; i < n; ++i)
            a = fmaf(w[i], pb_value(pv[(((pb_i64)table[i / PB_PS] * PB_H + kvh) * PB_PS + i % PB_PS) * PB_D + d]), a);
        out[row * PB_D + d] = a;
    }
}

extern "C" __global__ void __launch_bounds__(256) pb_attend_scores(
    const float* weights, const int* lengths, const float* scores, float* out, pb_i64 longest, pb_i64 ns, int group) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_u32 blocks = (pb_u32)((longest + 255) / 256);
    const pb_i64 i = (pb_i64)(blockIdx.x % blocks) * 256 + threadIdx.x, row = blockIdx.x / blocks;
    if (i >= longest) return;
    float a = 0.0f;
    if (i < lengths[row / PB_H]) {
        a = i < ns ? scores[row * ns + i] : 0.0f;
        for (int g = 0; g < group; ++g) a += weights[(row * group + g) * longest + i];
    }
    out[row * longest + i] = a;
}
)PB";
        }

        std::string defines(int64_t heads, int64_t dim, int64_t page, bool bf16) {
            std::ostringstream os;
            os << "#define PB_H " << heads << "\n#define PB_D " << dim << "\n#define PB_PS " << page
               << "\n#define PB_BF16 " << (bf16 ? 1 : 0) << "\n";
            return os.str();
        }

        op_kernel& kernel_of(const char* name, const std::string& defs) {
            return op_kernel_for(std::string{name} + "\n" + defs, [&](op_kernel& k) {
                k.name = name;
                k.source = std::string{kernel_prelude()} + defs + device_source();
            });
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
        expect(std::isfinite(scale), "paged_attention: scale must be finite");
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
        op_operand x = operand(q, stream, false), xs;
        if (scores != nullptr) xs = operand(*scores, stream, false);
        op_result out = new_result(shape, device, stream);
        order_read(*cuda_jit::buffer_access::state(batch.data), stream);
        order_read(*cuda_jit::buffer_access::state(c.k), stream);
        order_read(*cuda_jit::buffer_access::state(c.v), stream);
        const std::string defs = defines(c.heads, c.dim, c.page_size, c.type == cache_type::bf16);
        int64_t longest = batch.longest;
        int heads = static_cast<int>(shape[1]), group = static_cast<int>(shape[1] / c.heads);
        int width = static_cast<int>(batch.table_width);
        auto scratch = allocate(device, static_cast<size_t>(std::max<int64_t>(1, n * heads * longest)) * sizeof(float), stream);
        uint64_t weights = address(scratch), pk = address(c.k), pv = address(c.v);
        void* params[] = {&x.ptr, &pk,      &pv,    &batch.lengths_at, &batch.tables_at, &weights,
                          &out.ptr, &longest, &width, &heads,          &group,           &scale};
        op_launch(kernel_of("pb_attend", defs), device, stream, {static_cast<uint32_t>(n * heads), 1, 1}, 256, params);
        std::vector<tensor> results;
        results.push_back(finish(std::move(out)));
        if (scored) {
            op_result os = new_result({n, c.heads, longest}, device, stream);
            if (longest != 0) {
                void* sparams[] = {&weights, &batch.lengths_at, &xs.ptr, &os.ptr, &longest, &ns, &group};
                const int64_t blocks = (longest + 255) / 256 * n * c.heads;
                expect(blocks <= 0x7fffffff, "paged_attention_scored: too many slots");
                op_launch(kernel_of("pb_attend_scores", defs), device, stream, {static_cast<uint32_t>(blocks), 1, 1},
                          256, sparams);
            }
            results.push_back(finish(std::move(os)));
        }
        return results;
    }

    void paged_attention_sources(kernel_list& out) {
        for (const bool bf16 : {true, false})
            out.emplace_back(std::string{"pb_attend_"} + (bf16 ? "bf16" : "f32"),
                             std::string{kernel_prelude()} + defines(8, 128, 64, bf16) + device_source());
    }

} // namespace porch::detail
