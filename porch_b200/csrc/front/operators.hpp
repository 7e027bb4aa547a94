// Eager operators of a transformer's decode step (norms and rotation of
// query and key heads, a paged key/value cache, its attention, its eviction and
// its reading, log probabilities of tokens and their gradient). They have no counterpart in the reference, whose graphs end at
// matmul and softmax; each takes realised tensors (a lazy one is realised
// first), enqueues its kernels on the calling thread's stream and returns
// realised tensors, as allgather_rows does.
#pragma once

#include "lower.hpp"

#include <array>
#include <atomic>
#include <functional>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

namespace porch::detail {

    // ------------------------------------------------------------ launches --
    // One NVRTC instantiation of an operator's kernel source: compiled once
    // per process for its constants, loaded once per device.
    struct op_kernel {
        std::string name;
        std::string source;
        uint32_t smem = 0;
        uint64_t image_key = 0;
        std::mutex mutex;
        std::array<std::atomic<pbrt_function>, 16> function{};

        pbrt_function on(int device); // loaded by the first call
    };

    // The kernel for `key` (its name's address and every constant of its
    // source), made by `make` the first time.
    using op_key = std::array<int64_t, 12>;
    op_kernel& op_kernel_for(const op_key& key, const std::function<void(op_kernel&)>& make);

    // Launches `k` on `stream` so that it overlaps the previous kernel's tail:
    // every kernel here executes griddepcontrol.wait before it reads or writes
    // what other kernels do. What comes before the wait (attention's and its
    // join's plan, lengths and tables) is only ever written by an upload that
    // the host has waited for, never by a kernel.
    void op_launch(op_kernel& k, int device, const std::shared_ptr<stream_ref>& stream,
                   std::array<uint32_t, 3> grid, uint32_t threads, void** params, uint32_t cluster = 1);

    int sm_count(int device);

    // ------------------------------------------------------------ operands --
    // A float32 operand read in place: device address of element 0 and its
    // strides (a strided view is not copied as long as its innermost axis is
    // contiguous; otherwise, and unless `strided`, it is made contiguous and
    // only its address is filled in). Ordered behind its producer on `stream`.
    struct op_operand {
        std::shared_ptr<realized_storage> storage;
        uint64_t ptr = 0;
        std::vector<index_t> shape;
        std::vector<index_t> strides;
        int device = 0;
    };

    // Shape and device checks come first and need no device; operand() then
    // realises.
    std::vector<index_t> shape_of(const tensor& t);
    bool has_shape(const tensor& t, std::initializer_list<index_t> shape);
    // Throws for placeholders: they have no address.
    op_operand operand(const tensor& t, const std::shared_ptr<stream_ref>& stream, bool strided);
    // The device that `t`'s values live on; throws for placeholders.
    int device_of(const tensor& t, const char* what);
    // The widest of 4, 2, 1 floats at which every row of `x` can be loaded.
    int vector_width(const op_operand& x);

    // A new realised tensor whose block belongs to `stream`.
    struct op_result {
        std::shared_ptr<realized_storage> storage;
        std::vector<index_t> shape;
        uint64_t ptr = 0;
    };
    op_result new_result(std::vector<index_t> shape, int device, const std::shared_ptr<stream_ref>& stream);
    tensor finish(op_result&& r);

    inline uint64_t address(const cuda_jit::device_buffer& b) {
        const auto& st = cuda_jit::buffer_access::state(b);
        return st == nullptr ? 0 : st->ptr;
    }

    // Makes `stream` wait for what is enqueued on `first` so far.
    void order_behind(const std::shared_ptr<stream_ref>& first, const std::shared_ptr<stream_ref>& stream);

    // Makes `stream` wait for everything that reads or wrote the buffer on
    // other streams and then owns it: called before a kernel writes in place.
    void order_write(cuda_jit::device_buffer_state& buffer, const std::shared_ptr<stream_ref>& stream);

    // --------------------------------------------------------------- norms --
    struct norm_rope_args {
        const tensor* q = nullptr;
        const tensor* k = nullptr;
        const tensor* q_weight = nullptr;
        const tensor* k_weight = nullptr;
        const tensor* cos = nullptr;
        const tensor* sin = nullptr;
        const tensor* positions = nullptr;
        float eps = 1e-6F;
        bool interleaved = false;
    };
    std::array<tensor, 2> qk_norm_rope(const norm_rope_args& a);
    std::array<tensor, 4> qk_norm_rope_backward(const tensor& dq, const tensor& dk, const norm_rope_args& a);

    // ------------------------------------------------------ log probabilities --
    // {log probabilities, entropies, norms}, and where `top` is not 0 the
    // alternatives' log probabilities and tokens.
    std::vector<tensor> token_logprobs(const tensor& logits, const tensor& tokens, int64_t top);
    // The logits' gradient; d_entropy and entropy both or neither.
    tensor token_logprobs_backward(const tensor& d_said, const tensor& logits, const tensor& tokens, const tensor& norm,
                                   const tensor* d_entropy, const tensor* entropy);

    // --------------------------------------------------------------- cache --
    enum class cache_type : int { f32 = 0, bf16 = 1, i8 = 3 };

    // How the last attention over a cache shared out its work, for which the
    // next batch prepares its plan: with the upload that the batch waits for
    // anyway, instead of one that the step's first attention would wait for.
    struct plan_hint {
        std::mutex mutex;
        int64_t chunks = 0, ctas = 0; // 0: none yet
        int64_t group = 0;            // query heads of a key head, of the last shared prefix
    };

    // Pools of pages of keys and values: [pages, heads, page_size, dim], so
    // the rows of one page and head are one contiguous block. An 8-bit pool has
    // its rows' scales, [pages, heads, page_size], behind the codes.
    struct kv_cache {
        int64_t pages = 0, page_size = 0, heads = 0, dim = 0;
        cache_type type = cache_type::f32;
        int device = 0;
        cuda_jit::device_buffer k, v;
        // Held from a call's ordering on the pools until its last kernel on
        // them is enqueued: the order of calls from several threads is the
        // order of their kernels. Kernels are compiled and memory is allocated
        // before it is taken.
        std::mutex order;
        std::shared_ptr<plan_hint> hint = std::make_shared<plan_hint>();
        int width() const { return type == cache_type::f32 ? 4 : (type == cache_type::bf16 ? 2 : 1); } // bytes of a value
        int64_t values_bytes() const { return pages * heads * page_size * dim * width(); } // of one pool, without scales
        // TMA maps of both pools as [rows, dim]: boxes of 128 bytes by a page,
        // or by 64 rows of a larger one.
        struct alignas(64) tensor_map {
            unsigned char bytes[128];
        } map_k, map_v;
    };
    std::shared_ptr<kv_cache> make_cache(int64_t pages, int64_t page_size, int64_t heads, int64_t dim,
                                         cache_type type, int device);

    // The calling thread's stream, made to wait for what was called on the cache.
    pbrt_stream cache_ordered(kv_cache& c);

    // How attention's CTAs share a batch's slots, uploaded.
    struct batch_plan {
        int64_t chunks = 1; // query heads of a key head come in this many rows
        int64_t limit = 0;  // CTAs asked for
        int64_t ctas = 0, working = 0; // working: those that have tiles; the others clear empty rows
        int64_t joins = 0, most_parts = 0;
        cuda_jit::device_buffer data; // 16 bytes per CTA, then 16 per row to join
    };
    // The same for sequences that share a prefix. Rows are runs of slots of one
    // key head with the queries that read them: the prefixes' first, then what
    // follows them in each sequence.
    struct shared_plan {
        int64_t group = 0; // query heads of a key head
        // One launch's rows. The prefixes have one of their own where the tensor
        // cores' large tiles take them (else the second has them, too).
        struct stage {
            int per = 8; // queries that a row holds
            int64_t ctas = 0, parts = 0;
            uint64_t rows_at = 0, work_at = 0; // device addresses
        };
        stage prefix, rest;
        int64_t most_parts = 0, units = 0; // units: of the join
        cuda_jit::device_buffer data;
        uint64_t parts_at = 0, outs_at = 0, units_at = 0;
    };
    struct batch_plans {
        std::shared_ptr<plan_hint> hint; // of the cache that the batch was made for
        std::mutex mutex;
        std::vector<std::unique_ptr<batch_plan>> made;
        std::vector<std::unique_ptr<shared_plan>> shared;
    };

    // The sequences of one step: page tables, slots in use and the rows that
    // the step's new tokens go to, checked on the host and uploaded once for
    // every layer and call of the step.
    struct kv_batch {
        std::shared_ptr<kv_cache> cache;
        std::vector<int64_t> lengths;
        std::vector<int64_t> newest;   // position of each sequence's newest slot
        int64_t longest = 0, tokens = 0, slots = 0; // tokens: new ones, slots: all, over all sequences
        int64_t table_width = 0;
        bool shared_pages = false;       // a page serves two sequences, or one twice
        // Sequences next to each other whose first `slots` slots are the same pages.
        struct group {
            int64_t first = 0, members = 0, slots = 0;
        };
        std::vector<group> groups;
        bool always_share = false;       // whatever they spare: made while the test hook was on
        cuda_jit::device_buffer data;    // int32: lengths, newest, tables, then 8-byte rows and starts
        // Made once with the batch for the number of query heads that its cache
        // last saw (up to 8 for each key head until then), and by the first
        // call that needs another.
        std::shared_ptr<batch_plans> plans = std::make_shared<batch_plans>();
        // Device addresses. starts: the slots of all sequences before each, and of all.
        uint64_t lengths_at = 0, newest_at = 0, tables_at = 0, rows_at = 0, starts_at = 0;
        int64_t sequences() const { return static_cast<int64_t>(lengths.size()); }
    };
    std::shared_ptr<kv_batch> make_batch(std::shared_ptr<kv_cache> cache, const int32_t* tables, size_t sequences,
                                         size_t width, const int64_t* lengths, const int64_t* appended,
                                         const int64_t* newest, const int64_t* prefix = nullptr);

    // The plan for this many chunks and CTAs, which the cache's next batch gets.
    const batch_plan& plan_of(kv_batch& batch, int64_t chunks, int64_t ctas);
    // The plan that a new batch begins with.
    void prepare_plan(kv_batch& batch);
    // How many CTAs of an SM a plan for `group` query heads of each key head
    // counts on, and the bytes of shared memory that each takes.
    std::pair<int, int> attention_shape(int64_t dim, cache_type type, int64_t group);
    // Test hook (0: off): block 0 of an attention never gets its tiles, so its
    // bounded waits expire (1), or gives up while its first ones are on their
    // way (2).
    void set_test_attention_stall(int mode);
    // Test hook: of batches made while it is on, prefixes are worked through once
    // whatever their size.
    void set_test_share_prefix(bool on);
    bool test_share_prefix();
    // The plan as text ("work <row> <tile> <tiles>" per CTA, "join <row>
    // <first CTA> <parts> <place>" per row), without a device.
    std::string attention_schedule(const std::vector<int64_t>& lengths, int64_t heads, int64_t chunks, int64_t ctas,
                                   int64_t dim, cache_type type);

    // The same sequences over another cache of the same shape; shares the upload.
    std::shared_ptr<kv_batch> batch_on(const kv_batch& batch, std::shared_ptr<kv_cache> cache);

    // Writes the step's new keys and values, [tokens, heads, dim], into their rows.
    void cache_append(kv_batch& batch, const tensor& k, const tensor& v);
    // {keys, values} of every slot in use, [slots of all sequences, heads, dim].
    std::array<tensor, 2> cache_read(kv_batch& batch);
    // {attention, new scores} (the second only when `scored`).
    std::vector<tensor> paged_attention(const tensor& q, kv_batch& batch, float scale, bool scored,
                                        const tensor* scores);
    std::array<tensor, 2> cache_evict(kv_batch& batch, const tensor& scores, const tensor* positions,
                                      int64_t budget, int64_t recent, int64_t sinks);

    // Sources of representative instantiations of every operator kernel, in
    // the "kernel <name> ..." format of describe_plan, for build checks.
    std::string operator_sources();
    using kernel_list = std::vector<std::pair<std::string, std::string>>;
    void norm_rope_sources(kernel_list& out);
    void token_logprobs_sources(kernel_list& out);
    void paged_cache_sources(kernel_list& out);
    void paged_attention_sources(kernel_list& out);
    void prefix_attention_sources(kernel_list& out);

    // Whether there is a kernel of 128 queries a row for prefixes in this cache
    // (bfloat16, head_dim up to 128), and that kernel: 384 threads, a CTA an SM;
    // `wide`: every query's row starts on 16 bytes.
    bool prefix_attention_takes(const kv_cache& c);
    op_kernel& prefix_attention_kernel(const kv_cache& c, bool wide, int stall);

} // namespace porch::detail
