// porch::cuda_jit public API (include/porch/cuda_jit.hpp) and the stream /
// buffer plumbing used by the front-end, on top of the runtime C-ABI.
//
// Differences from the reference's src/cuda_jit.cpp that matter on B200:
//  - cross-stream dependencies are stream waits on events, not host
//    synchronisations of the producer stream (src/cuda_jit.cpp:809-813);
//  - a buffer's stream-ordered free is ordered after every foreign reader;
//  - PTX given to launch_* is loaded once per (device, image) instead of
//    cuModuleLoadData on every launch (src/cuda_jit.cpp:819-823).
#include "detail.hpp"

#include <algorithm>
#include <cstring>
#include <map>
#include <sstream>
#include <stdexcept>
#include <unordered_map>

namespace porch::detail {

    [[noreturn]] void throw_status(int status) {
        std::string message = pbrt_last_error();
        switch (status) {
            case PBRT_ERR_INVALID:
                throw std::invalid_argument(message);
            case PBRT_ERR_RANGE:
                throw std::out_of_range(message);
            case PBRT_ERR_COMPILE:
                throw cuda_jit::compilation_error(message);
            default:
                throw std::runtime_error(message);
        }
    }

    stream_ref::~stream_ref() {
        if (stream == nullptr) return;
        (void)pbrt_stream_synchronize(device, stream);
        (void)pbrt_stream_destroy(device, stream);
    }

    namespace {
        struct thread_stream_table {
            std::vector<std::shared_ptr<stream_ref>> streams;
        };
        thread_local thread_stream_table tl_streams;
        thread_local thread_stream_table tl_upload_streams;
        thread_local thread_stream_table tl_side_streams;

        std::shared_ptr<stream_ref> stream_in(thread_stream_table& t, int device) {
            auto& table = t.streams;
            if (device < 0)
                throw std::invalid_argument("CUDA device ordinal must be non-negative");
            if (table.size() <= static_cast<size_t>(device))
                table.resize(static_cast<size_t>(device) + 1);
            std::shared_ptr<stream_ref>& slot = table[static_cast<size_t>(device)];
            if (slot == nullptr) {
                pbrt_stream s = nullptr;
                check(pbrt_stream_create(device, &s));
                slot = std::make_shared<stream_ref>(device, s);
            }
            return slot;
        }
    } // namespace

    std::shared_ptr<stream_ref> upload_stream(int device) { return stream_in(tl_upload_streams, device); }
    std::shared_ptr<stream_ref> side_stream(int device) { return stream_in(tl_side_streams, device); }

    std::shared_ptr<stream_ref> current_stream(int device) {
        auto& table = tl_streams.streams;
        if (device < 0)
            throw std::invalid_argument("CUDA device ordinal must be non-negative");
        if (table.size() <= static_cast<size_t>(device))
            table.resize(static_cast<size_t>(device) + 1);
        std::shared_ptr<stream_ref>& slot = table[static_cast<size_t>(device)];
        if (slot == nullptr) {
            pbrt_stream s = nullptr;
            check(pbrt_stream_create(device, &s));
            slot = std::make_shared<stream_ref>(device, s);
        }
        return slot;
    }

    std::vector<std::shared_ptr<stream_ref>> thread_streams() {
        std::vector<std::shared_ptr<stream_ref>> out;
        for (const auto& s : tl_streams.streams)
            if (s != nullptr) out.push_back(s);
        for (const auto& s : tl_upload_streams.streams)
            if (s != nullptr) out.push_back(s);
        return out;
    }

    // ------------------------------------------------- caching allocator --
    // Freed blocks are kept per device in size classes together with the
    // stream that produced them; a request on that same stream reuses one
    // with no driver call (stream order already makes it safe). A block also
    // read on other streams waits in a pending list with an event recorded
    // on each of those readers, and joins its producer stream's free list
    // once every event has completed: no stream is ever made to wait for
    // another, so a reader (a gather on a communicator's stream) overlaps
    // the producer's next work. On allocation failure every cached block of
    // the device (pending ones after their readers finish) is returned to
    // the driver and the request retried once.
    namespace {
        struct cached_block {
            uint64_t ptr;
            std::shared_ptr<stream_ref> stream;
        };

        struct pending_block {
            uint64_t ptr;
            size_t capacity;
            std::shared_ptr<stream_ref> stream;
            std::vector<std::pair<int, pbrt_event>> events; // (device, event) per foreign reader
        };

        // Blocks are carved from slabs of device memory by bumping an
        // offset, so a cache miss costs no driver call: cuMemAlloc runs once
        // per 256 MiB slab (a larger request gets a slab of its own), and it
        // stalls behind the device's queued work, up to milliseconds while
        // GEMMs run. A block is never handed back to its slab one by one: it
        // lives in the size-class free lists; a slab returns to the driver
        // once every block carved from it has been dropped from the cache.
        struct slab {
            size_t size = 0;
            size_t used = 0; // bump offset
            size_t live = 0; // blocks carved and not yet dropped
        };
        constexpr size_t kSlabBytes = size_t{256} << 20;

        struct device_cache {
            std::mutex mutex;
            std::unordered_map<size_t, std::vector<cached_block>> free;
            std::vector<pending_block> pending;
            size_t cached_bytes = 0;
            std::map<uint64_t, slab> slabs; // by base address
            uint64_t current = 0;           // the slab new blocks are bumped from
        };

        // A block of `cls` bytes (a multiple of 512) from the current slab,
        // or from a new one. Caller holds dc.mutex.
        int slab_alloc_locked(int device, device_cache& dc, size_t cls, uint64_t* out) {
            if (dc.current != 0) {
                slab& s = dc.slabs.at(dc.current);
                if (s.used + cls <= s.size) {
                    *out = dc.current + s.used;
                    s.used += cls;
                    ++s.live;
                    return PBRT_OK;
                }
            }
            const size_t size = std::max(kSlabBytes, cls);
            uint64_t base = 0;
            const int st = pbrt_mem_alloc(device, size, &base);
            if (st != PBRT_OK) return st;
            host_count("slab_alloc");
            dc.slabs[base] = slab{size, cls, 1};
            if (size == kSlabBytes) dc.current = base; // larger slabs hold one block
            *out = base;
            return PBRT_OK;
        }

        // Drops one block carved from a slab; the slab goes back to the
        // driver when it was the last (cuMemFree waits for the device's
        // queued work, so nothing still running can touch it). Caller holds
        // dc.mutex.
        void slab_drop_locked(int device, device_cache& dc, uint64_t ptr) {
            auto it = dc.slabs.upper_bound(ptr);
            if (it == dc.slabs.begin()) return;
            --it;
            if (ptr >= it->first + it->second.size) return;
            if (--it->second.live != 0) return;
            (void)pbrt_mem_free(device, it->first);
            if (dc.current == it->first) dc.current = 0;
            dc.slabs.erase(it);
        }

        // Moves pending blocks whose readers have all finished to the free
        // lists. Caller holds dc.mutex.
        void reap_locked(device_cache& dc) {
            for (size_t i = 0; i < dc.pending.size();) {
                pending_block& p = dc.pending[i];
                bool done = true;
                for (const auto& [dev, ev] : p.events) {
                    int d = 0;
                    if (pbrt_event_query(dev, ev, &d) != PBRT_OK || d == 0) {
                        done = false;
                        break;
                    }
                }
                if (!done) {
                    ++i;
                    continue;
                }
                for (const auto& [dev, ev] : p.events) (void)pbrt_event_destroy(dev, ev);
                dc.free[p.capacity].push_back({p.ptr, std::move(p.stream)});
                dc.cached_bytes += p.capacity;
                dc.pending[i] = std::move(dc.pending.back());
                dc.pending.pop_back();
            }
        }

        struct block_cache {
            std::mutex mutex;
            std::vector<std::unique_ptr<device_cache>> devices;
            device_cache& of(int device) {
                std::scoped_lock lock{mutex};
                if (devices.size() <= static_cast<size_t>(device))
                    devices.resize(static_cast<size_t>(device) + 1);
                auto& d = devices[static_cast<size_t>(device)];
                if (!d) d = std::make_unique<device_cache>();
                return *d;
            }
        };

        block_cache& blocks() {
            static block_cache* c = new block_cache(); // lives until exit
            return *c;
        }

        size_t size_class(size_t bytes) {
            if (bytes <= (size_t{1} << 20)) return (bytes + 511) & ~size_t{511};
            return (bytes + (size_t{2} << 20) - 1) & ~((size_t{2} << 20) - 1);
        }
    } // namespace

    size_t release_cached_blocks(int device) {
        device_cache& dc = blocks().of(device);
        std::unordered_map<size_t, std::vector<cached_block>> drop;
        std::vector<pending_block> waiting;
        size_t bytes = 0;
        {
            std::scoped_lock lock{dc.mutex};
            drop.swap(dc.free);
            waiting.swap(dc.pending);
            bytes = dc.cached_bytes;
            dc.cached_bytes = 0;
        }
        for (auto& p : waiting) {
            for (const auto& [dev, ev] : p.events) {
                (void)pbrt_event_synchronize(dev, ev);
                (void)pbrt_event_destroy(dev, ev);
            }
            bytes += p.capacity;
        }
        // Slabs whose every block is dropped here go back to the driver.
        std::scoped_lock lock{dc.mutex};
        for (auto& [size, list] : drop)
            for (auto& b : list) slab_drop_locked(device, dc, b.ptr);
        for (auto& p : waiting) slab_drop_locked(device, dc, p.ptr);
        return bytes;
    }

    void release_block(int device, uint64_t ptr, size_t capacity) {
        if (capacity == 0) {
            (void)pbrt_mem_free(device, ptr);
            return;
        }
        device_cache& dc = blocks().of(device);
        std::scoped_lock lock{dc.mutex};
        slab_drop_locked(device, dc, ptr);
    }

    void defer_recycle(int device, uint64_t ptr, size_t capacity, std::shared_ptr<stream_ref> stream,
                       std::vector<std::pair<int, pbrt_event>> events) {
        device_cache& dc = blocks().of(device);
        std::scoped_lock lock{dc.mutex};
        dc.pending.push_back({ptr, capacity, std::move(stream), std::move(events)});
    }

    cuda_jit::device_buffer allocate(
        int device, size_t bytes, const std::shared_ptr<stream_ref>& stream
    ) {
        auto state = std::make_shared<cuda_jit::device_buffer_state>();
        state->device = device;
        state->bytes = bytes;
        if (bytes != 0) {
            const size_t cls = size_class(bytes);
            state->capacity = cls;
            device_cache& dc = blocks().of(device);
            {
                std::scoped_lock lock{dc.mutex};
                if (!dc.pending.empty()) reap_locked(dc);
                auto it = dc.free.find(cls);
                if (it != dc.free.end()) {
                    auto& list = it->second;
                    for (size_t i = list.size(); i > 0; --i) {
                        if (list[i - 1].stream == stream) {
                            state->ptr = list[i - 1].ptr;
                            list.erase(list.begin() + static_cast<ptrdiff_t>(i - 1));
                            dc.cached_bytes -= cls;
                            break;
                        }
                    }
                }
            }
            host_count(state->ptr ? "alloc_cache_hit" : "alloc_cache_miss");
            if (state->ptr == 0) {
                int st = PBRT_OK;
                {
                    std::scoped_lock lock{dc.mutex};
                    st = slab_alloc_locked(device, dc, cls, &state->ptr);
                }
                if (st != PBRT_OK && release_cached_blocks(device) != 0) {
                    std::scoped_lock lock{dc.mutex};
                    st = slab_alloc_locked(device, dc, cls, &state->ptr);
                }
                check(st);
            }
            state->producer = stream;
        }
        return cuda_jit::buffer_access::wrap(std::move(state));
    }

    void recycle(int device, uint64_t ptr, size_t capacity, std::shared_ptr<stream_ref> stream) {
        device_cache& dc = blocks().of(device);
        std::scoped_lock lock{dc.mutex};
        dc.free[capacity].push_back({ptr, std::move(stream)});
        dc.cached_bytes += capacity;
    }

    void order_read(
        cuda_jit::device_buffer_state& buffer,
        const std::shared_ptr<stream_ref>& stream
    ) {
        std::shared_ptr<stream_ref> producer;
        {
            std::scoped_lock lock{buffer.mutex};
            producer = buffer.producer;
            if (producer == nullptr || producer == stream) return;
            host_count("order_read_cross_stream");
            bool known = false;
            for (const auto& r : buffer.readers) known = known || r == stream;
            if (!known) buffer.readers.push_back(stream);
        }
        if (producer->device == stream->device && buffer.ready != nullptr) {
            // Recorded right after the buffer's own upload: later work on the
            // producer stream (other uploads) is not waited for.
            check(pbrt_stream_wait_event(stream->device, stream->stream, buffer.ready));
        } else if (producer->device == stream->device) {
            pbrt_event e = nullptr;
            check(pbrt_event_create(producer->device, 0, &e));
            check(pbrt_event_record(producer->device, e, producer->stream));
            check(pbrt_stream_wait_event(stream->device, stream->stream, e));
            (void)pbrt_event_destroy(producer->device, e);
        } else {
            // Different devices: the reader copies or loads over NVLink; keep
            // it simple and exact by draining the producer first.
            check(pbrt_stream_synchronize(producer->device, producer->stream));
        }
    }

    void set_producer(
        cuda_jit::device_buffer_state& buffer, std::shared_ptr<stream_ref> stream
    ) {
        std::scoped_lock lock{buffer.mutex};
        buffer.producer = std::move(stream);
    }

} // namespace porch::detail

namespace porch::cuda_jit {

    device_buffer_state::~device_buffer_state() {
        if (ready != nullptr) (void)pbrt_event_destroy(device, ready);
        if (ptr == 0) return;
        try {
            std::shared_ptr<detail::stream_ref> free_stream =
                producer != nullptr ? producer : detail::current_stream(device);
            bool foreign = false;
            for (const auto& reader : readers) foreign = foreign || reader != free_stream;
            if (!foreign && capacity != 0) {
                // Only this stream ever touched it: keep it for reuse.
                detail::recycle(device, ptr, capacity, std::move(free_stream));
                return;
            }
            // Read on other streams: an event behind each of those reads;
            // the block rejoins the producer stream's free list once they
            // have all completed (the producer's own later reads are ordered
            // by its stream). Nothing waits now.
            std::vector<std::pair<int, pbrt_event>> events;
            bool ok = true;
            for (const auto& reader : readers) {
                if (reader == free_stream) continue;
                pbrt_event e = nullptr;
                if (pbrt_event_create(reader->device, 0, &e) != PBRT_OK) {
                    ok = false;
                    break;
                }
                events.emplace_back(reader->device, e);
                if (pbrt_event_record(reader->device, e, reader->stream) != PBRT_OK) {
                    ok = false;
                    break;
                }
            }
            if (ok && capacity != 0) {
                detail::defer_recycle(device, ptr, capacity, std::move(free_stream), std::move(events));
                return;
            }
            // No events: drain the readers on the host, then free (cuMemFree
            // also waits for the producer's queued work).
            for (const auto& [dev, ev] : events) (void)pbrt_event_destroy(dev, ev);
            for (const auto& reader : readers)
                if (reader != free_stream) (void)pbrt_stream_synchronize(reader->device, reader->stream);
            detail::release_block(device, ptr, capacity);
        } catch (...) {
        }
    }

    device_buffer::device_buffer(size_t bytes) {
        if (bytes == 0) return;
        *this = detail::allocate(0, bytes, detail::current_stream(0));
    }

    bool device_buffer::empty() const noexcept {
        return state_ == nullptr || state_->bytes == 0;
    }

    size_t device_buffer::size_bytes() const noexcept {
        return state_ == nullptr ? 0 : state_->bytes;
    }

    compilation_error::compilation_error(std::string log)
        : std::runtime_error(log), log_(std::move(log)) {}

    const std::string& compilation_error::log() const noexcept { return log_; }

    bool is_available() noexcept { return pbrt_available() == 1; }

    std::string compile_to_ptx(
        std::string_view source, const std::vector<std::string>& options
    ) {
        std::vector<const char*> opts;
        opts.reserve(options.size());
        for (const std::string& o : options) opts.push_back(o.c_str());
        const std::string text{source};
        uint64_t key = 0;
        detail::check(pbrt_compile(text.c_str(), opts.empty() ? nullptr : opts.data(),
                                   static_cast<int>(opts.size()), 0, &key));
        const void* image = nullptr;
        size_t size = 0;
        detail::check(pbrt_compiled_image(key, &image, &size));
        std::string ptx(static_cast<const char*>(image), size);
        while (!ptx.empty() && ptx.back() == '\0') ptx.pop_back();
        return ptx;
    }

    namespace {
        void require_device_bytes(
            const device_buffer& buffer, size_t bytes, const char* name
        ) {
            if (buffer.size_bytes() < bytes)
                throw std::invalid_argument(
                    std::string{name} + " device buffer is too small"
                );
        }
    } // namespace

    device_buffer make_device_buffer(std::span<const float32_t> source) {
        device_buffer buffer{source.size_bytes()};
        copy_to_device(buffer, source);
        return buffer;
    }

    void copy_to_device(device_buffer& buffer, std::span<const float32_t> source) {
        if (source.empty()) return;
        require_device_bytes(buffer, source.size_bytes(), "target");
        device_buffer_state& st = *buffer.state_;
        auto stream = detail::current_stream(st.device);
        detail::order_read(st, stream);
        detail::check(pbrt_memcpy_h2d_async(st.device, st.ptr, source.data(),
                                            source.size_bytes(), stream->stream));
        // The source span may be pageable and short-lived: complete the copy
        // before returning, as the reference does (src/cuda_jit.cpp:729-732).
        detail::check(pbrt_stream_synchronize(st.device, stream->stream));
        detail::set_producer(st, stream);
    }

    void copy_to_host(const device_buffer& buffer, std::span<float32_t> target) {
        if (target.empty()) return;
        require_device_bytes(buffer, target.size_bytes(), "source");
        device_buffer_state& st = *buffer.state_;
        auto stream = detail::current_stream(st.device);
        detail::order_read(st, stream);
        detail::check(pbrt_memcpy_d2h_async(st.device, target.data(), st.ptr,
                                            target.size_bytes(), stream->stream));
        detail::check(pbrt_stream_synchronize(st.device, stream->stream));
        int code = 0;
        detail::check(pbrt_error_check(st.device, stream->stream, &code));
    }

    void synchronize() {
        // Drain this thread's streams on every device it has used (the
        // reference has one device and syncs its one thread-local stream,
        // src/cuda_jit.cpp:761).
        for (const auto& stream : detail::thread_streams()) {
            detail::check(pbrt_stream_synchronize(stream->device, stream->stream));
            int code = 0;
            detail::check(pbrt_error_check(stream->device, stream->stream, &code));
        }
    }

    namespace {
        // User-supplied PTX launch (drop-in for the reference's launch_*,
        // src/cuda_jit.cpp:789-948): same grid conventions, same checks.
        void launch_ptx(
            std::string_view ptx, std::string_view function,
            const std::vector<const device_buffer*>& inputs, device_buffer& out,
            size_t count, bool reduction
        ) {
            if (count == 0) return;
            const char* what = reduction ? "CUDA reduction input" : "CUDA elementwise input";
            for (const device_buffer* input : inputs) {
                if (input == nullptr) throw std::invalid_argument(std::string{what} + " is null");
                if (input->empty()) throw std::invalid_argument(std::string{what} + " is empty");
            }
            require_device_bytes(out, count * sizeof(float32_t), "out");
            device_buffer_state& ost = *buffer_access::state(out);
            const int device = ost.device;
            auto stream = detail::current_stream(device);
            for (const device_buffer* input : inputs)
                detail::order_read(*buffer_access::state(*input), stream);
            detail::order_read(ost, stream);

            const std::string text{ptx};
            uint64_t key = 0;
            detail::check(pbrt_register_image(text.c_str(), text.size() + 1, &key));
            pbrt_function fn = nullptr;
            const std::string name{function};
            detail::check(pbrt_get_function(device, key, name.c_str(), &fn));

            std::vector<uint64_t> ptrs;
            ptrs.reserve(inputs.size());
            for (const device_buffer* input : inputs) ptrs.push_back(buffer_access::state(*input)->ptr);
            uint64_t out_ptr = ost.ptr;
            uint64_t n = count;
            std::vector<void*> params;
            for (uint64_t& p : ptrs) params.push_back(&p);
            params.push_back(&out_ptr);
            params.push_back(&n);
            const uint32_t block[3] = {256, 1, 1};
            const uint32_t grid[3] = {
                reduction ? static_cast<uint32_t>(count)
                          : static_cast<uint32_t>((count + 255) / 256),
                1, 1};
            detail::check(pbrt_launch(device, fn, grid, block, 0, stream->stream,
                                      params.data(), nullptr));
            detail::set_producer(ost, stream);
        }
    } // namespace

    void launch_elementwise_binary(
        std::string_view ptx, std::string_view function,
        std::span<const float32_t> lhs, std::span<const float32_t> rhs,
        std::span<float32_t> out
    ) {
        if (lhs.size() != rhs.size() || lhs.size() != out.size())
            throw std::invalid_argument("CUDA elementwise operands must match");
        device_buffer device_lhs = make_device_buffer(lhs);
        device_buffer device_rhs = make_device_buffer(rhs);
        device_buffer device_out{out.size_bytes()};
        launch_elementwise_binary(ptx, function, device_lhs, device_rhs, device_out,
                                  out.size());
        copy_to_host(device_out, out);
    }

    void launch_elementwise_binary(
        std::string_view ptx, std::string_view function, const device_buffer& lhs,
        const device_buffer& rhs, device_buffer& out, size_t count
    ) {
        std::vector<const device_buffer*> inputs{&lhs, &rhs};
        launch_ptx(ptx, function, inputs, out, count, false);
    }

    void launch_fused_elementwise(
        std::string_view ptx, std::string_view function,
        const std::vector<const device_buffer*>& inputs, device_buffer& out,
        size_t count
    ) {
        launch_ptx(ptx, function, inputs, out, count, false);
    }

    void launch_fused_reduction(
        std::string_view ptx, std::string_view function,
        const std::vector<const device_buffer*>& inputs, device_buffer& out,
        size_t count
    ) {
        launch_ptx(ptx, function, inputs, out, count, true);
    }

} // namespace porch::cuda_jit
