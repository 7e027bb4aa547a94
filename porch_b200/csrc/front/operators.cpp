// Shared plumbing of the eager operators: kernel instantiation and launch,
// operand access, results, in-place ordering.
#include "operators.hpp"

#include <algorithm>
#include <sstream>
#include <stdexcept>
#include <unordered_map>

namespace porch::detail {

    namespace {
        uint64_t compile(const std::string& source) {
            std::vector<const char*> options;
            for (const auto& o : kernel_options()) options.push_back(o.c_str());
            uint64_t key = 0;
            check(pbrt_compile(source.c_str(), options.data(), static_cast<int>(options.size()), 1, &key));
            return key;
        }
    } // namespace

    pbrt_function op_kernel::on(int device) {
        if (device < 0 || device >= static_cast<int>(function.size()))
            throw std::invalid_argument("device ordinal out of range");
        auto& slot = function[static_cast<size_t>(device)];
        pbrt_function f = slot.load(std::memory_order_acquire);
        if (f != nullptr) return f;
        std::scoped_lock lock{mutex};
        check(pbrt_get_function(device, image_key, name.c_str(), &f));
        // The default limit of 48 KB is on dynamic and static memory together.
        if (smem != 0) check(pbrt_function_set_max_dynamic_smem(f, static_cast<int>(smem)));
        slot.store(f, std::memory_order_release);
        return f;
    }

    namespace {
        struct key_hash {
            size_t operator()(const op_key& k) const {
                uint64_t h = 0xcbf29ce484222325ULL;
                for (const int64_t v : k) h = (h ^ static_cast<uint64_t>(v)) * 0x9e3779b97f4a7c15ULL;
                return h ^ (h >> 32);
            }
        };
    } // namespace

    op_kernel& op_kernel_for(const op_key& key, const std::function<void(op_kernel&)>& make) {
        // The table's lock is held for the lookup alone: a kernel compiles under
        // its own entry's, so that it holds up nobody but those who need it.
        struct entry {
            std::mutex mutex;
            std::unique_ptr<op_kernel> made;
            std::atomic<op_kernel*> ready{nullptr};
        };
        static std::mutex mutex;
        static auto* table = new std::unordered_map<op_key, std::unique_ptr<entry>, key_hash>(); // lives until exit
        entry* e = nullptr;
        {
            std::scoped_lock lock{mutex};
            auto& slot = (*table)[key];
            if (slot == nullptr) slot = std::make_unique<entry>();
            e = slot.get();
        }
        if (op_kernel* k = e->ready.load(std::memory_order_acquire)) return *k;
        std::scoped_lock lock{e->mutex};
        if (e->made == nullptr) {
            auto k = std::make_unique<op_kernel>();
            make(*k);
            k->image_key = compile(k->source);
            e->made = std::move(k); // one that failed is tried again
            e->ready.store(e->made.get(), std::memory_order_release);
        }
        return *e->made;
    }

    void op_launch(op_kernel& k, int device, const std::shared_ptr<stream_ref>& stream,
                   std::array<uint32_t, 3> grid, uint32_t threads, void** params, uint32_t cluster) {
        const uint32_t block[3] = {threads, 1, 1}, clusters[3] = {cluster, 1, 1};
        check(pbrt_launch_ex(device, k.on(device), grid.data(), block, k.smem, stream->stream, params,
                             cluster > 1 ? clusters : nullptr, PBRT_LAUNCH_PDL));
    }

    int sm_count(int device) {
        static std::array<std::atomic<int>, 16> counts{};
        if (device < 0 || device >= 16) throw std::invalid_argument("device ordinal out of range");
        int n = counts[static_cast<size_t>(device)].load(std::memory_order_relaxed);
        if (n == 0) {
            check(pbrt_device_attribute(device, 16 /* multiprocessor count */, &n));
            counts[static_cast<size_t>(device)].store(n, std::memory_order_relaxed);
        }
        return n;
    }

    std::vector<index_t> shape_of(const tensor& t) { return {t.shape().begin(), t.shape().end()}; }

    bool has_shape(const tensor& t, std::initializer_list<index_t> shape) { return std::ranges::equal(t.shape(), shape); }

    int device_of(const tensor& t, const char* what) {
        auto s = tensor_access::storage(t);
        if (s->placeholder)
            throw std::runtime_error(std::string{what} + ": placeholder tensors hold no values");
        return s->device;
    }

    op_operand operand(const tensor& t, const std::shared_ptr<stream_ref>& stream, bool strided) {
        op_operand x;
        x.storage = tensor_access::storage(t);
        if (x.storage->placeholder) throw std::runtime_error("operands: placeholder tensors hold no values");
        if (strided) {
            x.shape = shape_of(t);
            x.strides = contiguous_strides(x.shape);
        }
        x.device = stream->device;
        if (x.storage->device != stream->device)
            throw std::invalid_argument("operands must live on one device");
        std::shared_ptr<realized_storage> base;
        strided_layout l;
        if (view_of(*x.storage, base, l)) {
            const bool inner = strided && !l.shape.empty() && l.shape == x.shape &&
                               (l.shape.back() <= 1 || l.strides.back() == 1);
            if (!inner) {
                make_contiguous(x.storage);
            } else {
                x.storage = base;
                x.strides = l.strides;
                x.ptr = static_cast<uint64_t>(l.offset) * sizeof(float32_t);
            }
        }
        const auto& st = cuda_jit::buffer_access::state(x.storage->device_values);
        if (st == nullptr || st->ptr == 0) {
            x.ptr = 0; // no elements
            return x;
        }
        order_read(*st, stream);
        x.ptr += st->ptr;
        return x;
    }

    int vector_width(const op_operand& x) {
        int w = 4;
        while (w > 1 && x.ptr % (static_cast<uint64_t>(w) * sizeof(float32_t)) != 0) w /= 2;
        for (size_t d = 0; d + 1 < x.strides.size(); ++d)
            if (x.shape[d] > 1)
                while (w > 1 && x.strides[d] % w != 0) w /= 2;
        return w;
    }

    op_result new_result(std::vector<index_t> shape, int device, const std::shared_ptr<stream_ref>& stream) {
        op_result r;
        r.storage = std::make_shared<realized_storage>();
        r.storage->count = checked_numel(shape);
        r.storage->device = device;
        r.storage->device_values = allocate(device, r.storage->count * sizeof(float32_t), stream);
        if (r.storage->count == 0) r.storage->host_current = true;
        r.ptr = address(r.storage->device_values);
        r.shape = std::move(shape);
        return r;
    }

    tensor finish(op_result&& r) {
        const device placement{r.storage->device};
        return tensor_access::from_storage(std::move(r.shape), std::move(r.storage), placement);
    }

    void order_write(cuda_jit::device_buffer_state& buffer, const std::shared_ptr<stream_ref>& stream) {
        std::vector<std::shared_ptr<stream_ref>> others;
        {
            std::scoped_lock lock{buffer.mutex};
            if (buffer.producer != nullptr && buffer.producer != stream) others.push_back(buffer.producer);
            for (const auto& r : buffer.readers)
                if (r != stream) others.push_back(r);
            buffer.readers.clear();
            buffer.producer = stream;
        }
        for (const auto& o : others) {
            pbrt_event e = nullptr;
            check(pbrt_event_create(o->device, 0, &e));
            int s = pbrt_event_record(o->device, e, o->stream);
            if (s == PBRT_OK) s = pbrt_stream_wait_event(stream->device, stream->stream, e);
            (void)pbrt_event_destroy(o->device, e);
            check(s);
        }
    }

    std::string operator_sources() {
        std::vector<std::pair<std::string, std::string>> all;
        norm_rope_sources(all);
        paged_cache_sources(all);
        paged_attention_sources(all);
        std::ostringstream os;
        for (const auto& [name, source] : all) (void)compile(source); // NVRTC takes it, too
        for (const auto& [name, source] : all) os << "kernel " << name << " : operator\n" << source << "\n";
        return os.str();
    }

} // namespace porch::detail
