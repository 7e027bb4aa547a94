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
// Thread: 8 values of one token's key or value. Bound by HBM: 4 B read and
// the cache's width written per value; a float32 value is rounded to nearest
// even bfloat16, the type that the cache holds.
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
static __device__ __forceinline__ pb_u32 pb_key(const pb_row& r, int i) {
    const float p = pb_place(r, i);
    return p > r.recent_from || p < r.sinks ? 0xffffffffu : pb_order(pb_score(r, i));
}

// Rank of this thread's flag among the block's 1024, and their number.
static __device__ __forceinline__ int pb_block_rank(bool flag, int* warps, int& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const pb_u32 votes = __ballot_sync(0xffffffffu, flag);
    __syncthreads();
    if (lane == 0) warps[w] = __popc(votes);
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < 32; ++i) {
        if (i < w) before += warps[i];
        total += warps[i];
    }
    return before + __popc(votes & ((1u << lane) - 1u));
}

// One block per sequence and key head: a radix select of the budget-th
// largest key (4 passes of 8 bits), then one pass in slot order that lists
// the free places below the budget and the kept slots past it.
extern "C" __global__ void __launch_bounds__(1024) pb_evict_select(
    const float* scores, const float* places, const int* lengths, const int* newest, float* out_scores,
    float* out_places, int* from, int* holes, pb_i64 ns, pb_i64 np, int budget, int recent, int sinks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ int hist[256];
    __shared__ int warps[32];
    __shared__ int chosen[2]; // digit, keys of it still wanted
    const pb_i64 row = blockIdx.x;
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
    int* map = from + row * budget;
    int* hole = holes + row * budget;
    for (int i = threadIdx.x; i < budget; i += 1024) map[i] = i;
    if (r.length > budget) {
        pb_u32 prefix = 0;
        int want = budget;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (threadIdx.x < 256) hist[threadIdx.x] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < r.length; i += 1024) {
                const pb_u32 key = pb_key(r, i);
                if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1);
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                int d = 255, left = want;
                while (hist[d] < left) left -= hist[d--];
                chosen[0] = d;
                chosen[1] = left;
            }
            __syncthreads();
            prefix |= (pb_u32)chosen[0] << shift;
            want = chosen[1];
            __syncthreads();
        }
        int ties = 0, nholes = 0, nlate = 0, total = 0;
        for (int base = 0; base < r.length; base += 1024) {
            const int i = base + threadIdx.x;
            const pb_u32 key = i < r.length ? pb_key(r, i) : 0u;
            const bool tie = i < r.length && key == prefix;
            const int rank = ties + pb_block_rank(tie, warps, total);
            ties += total;
            const bool kept = i < r.length && (key > prefix || (tie && rank < want));
            const int h = nholes + pb_block_rank(i < budget && !kept, warps, total);
            nholes += total;
            if (i < budget && !kept) hole[h] = i;
            __syncthreads(); // the list of places is complete below `base + 1024`
            const int l = nlate + pb_block_rank(i >= budget && kept, warps, total);
            nlate += total;
            if (i >= budget && kept) map[hole[l]] = i;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < budget; i += 1024) {
        const bool live = i < r.length;
        out_scores[row * budget + i] = live ? pb_score(r, map[i]) : 0.0f;
        out_places[row * budget + i] = live ? pb_place(r, map[i]) : -1.0f;
    }
}

// Warps copy the rows that moved, keys and values.
extern "C" __global__ void __launch_bounds__(256) pb_evict_move(
    char* pk, char* pv, const int* tables, const int* lengths, const int* from, pb_i64 rows, int width, int budget) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const pb_i64 id = ((pb_i64)blockIdx.x * 256 + threadIdx.x) / 32;
    const int lane = threadIdx.x & 31;
    if (id >= rows * budget) return;
    const pb_i64 row = id / budget;
    const int i = (int)(id - row * budget), src = from[id], s = (int)(row / PB_H), h = (int)(row % PB_H);
    if (src == i || i >= lengths[s]) return;
    const pb_i64 table = (pb_i64)s * width;
    const pb_i64 a = (((pb_i64)tables[table + src / PB_PS] * PB_H + h) * PB_PS + src % PB_PS) * PB_ROW;
    const pb_i64 b = (((pb_i64)tables[table + i / PB_PS] * PB_H + h) * PB_PS + i % PB_PS) * PB_ROW;
    for (int c = lane * 16; c < PB_ROW; c += 512) {
        *reinterpret_cast<uint4*>(pk + b + c) = *reinterpret_cast<const uint4*>(pk + a + c);
        *reinterpret_cast<uint4*>(pv + b + c) = *reinterpret_cast<const uint4*>(pv + a + c);
    }
}
)PB";
        }

        std::string defines(const kv_cache& c, bool wide) {
            std::ostringstream os;
            os << "#define PB_H " << c.heads << "\n#define PB_D " << c.dim << "\n#define PB_PS " << c.page_size
               << "\n#define PB_ROW " << c.dim * c.width() << "\n#define PB_BF16 " << (c.type == cache_type::bf16 ? 1 : 0)
               << "\n#define PB_WIDE " << (wide ? 1 : 0) << "\n";
            return os.str();
        }

        const char kAppend[] = "pb_cache_append";
        const char kSelect[] = "pb_evict_select";
        const char kMove[] = "pb_evict_move";

        op_kernel& kernel_of(const char* name, const kv_cache& c, bool wide = true) {
            const op_key key{reinterpret_cast<int64_t>(name), c.heads, c.dim, c.page_size, static_cast<int64_t>(c.type), wide};
            return op_kernel_for(key, [&](op_kernel& k) {
                k.name = name;
                k.source = std::string{kernel_prelude()} + defines(c, wide) + (name == kAppend ? append_source() : evict_source());
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
        return c;
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
        (void)plan_of(*b, 1, int64_t{attention_ctas_per_sm(*cache)} * sm_count(cache->device));
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
        order_read(*cuda_jit::buffer_access::state(batch.data), stream);
        order_write(*cuda_jit::buffer_access::state(c.k), stream);
        order_write(*cuda_jit::buffer_access::state(c.v), stream);
        uint64_t pk = address(c.k), pv = address(c.v);
        const int64_t blocks = (batch.tokens * c.heads * (c.dim / 8) + 255) / 256;
        expect(blocks <= 0x7fffffff, "cache_append: too many new tokens");
        void* params[] = {&xk.ptr,        &xv.ptr,        &pk,            &pv,            &batch.rows_at,
                          &batch.tokens,  &xk.strides[0], &xk.strides[1], &xv.strides[0], &xv.strides[1]};
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
        op_kernel& select = kernel_of(kSelect, c);
        op_kernel& move = kernel_of(kMove, c);
        int64_t rows = n * c.heads;
        auto scratch = allocate(device, static_cast<size_t>(rows * budget) * 2 * sizeof(int32_t), stream);
        uint64_t from = address(scratch), holes = from + static_cast<uint64_t>(rows * budget) * sizeof(int32_t);
        order_read(*cuda_jit::buffer_access::state(batch.data), stream);
        order_write(*cuda_jit::buffer_access::state(c.k), stream);
        order_write(*cuda_jit::buffer_access::state(c.v), stream);
        uint64_t pk = address(c.k), pv = address(c.v);
        int b = static_cast<int>(budget), rc = static_cast<int>(recent), sk = static_cast<int>(sinks);
        int width = static_cast<int>(batch.table_width);
        int64_t nsv = ns, npv = np;
        void* sparams[] = {&xs.ptr, &xp.ptr, &batch.lengths_at, &batch.newest_at, &os.ptr, &op.ptr, &from,
                           &holes,  &nsv,    &npv,              &b,               &rc,     &sk};
        op_launch(select, device, stream, {static_cast<uint32_t>(rows), 1, 1}, 1024, sparams);
        if (batch.longest > budget) {
            const int64_t blocks = (rows * budget + 7) / 8;
            expect(blocks <= 0x7fffffff, "cache_evict: too many rows");
            void* mparams[] = {&pk, &pv, &batch.tables_at, &batch.lengths_at, &from, &rows, &width, &b};
            op_launch(move, device, stream, {static_cast<uint32_t>(blocks), 1, 1}, 256, mparams);
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
        }
    }

} // namespace porch::detail
