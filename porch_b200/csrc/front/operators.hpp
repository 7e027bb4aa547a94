// Eager operators of a transformer's decode step (norms and rotation of
// query and key heads, a paged key/value cache, its attention and its
// eviction). They have no counterpart in the reference, whose graphs end at
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

        pbrt_function on(int device);
    };

    // The kernel for `key` (which spells out every constant of the source),
    // made by `make` the first time.
    op_kernel& op_kernel_for(const std::string& key, const std::function<void(op_kernel&)>& make);

    // Launches `k` on `stream`; every kernel here begins with
    // griddepcontrol.wait, so the launch overlaps the previous kernel's tail.
    void op_launch(op_kernel& k, int device, const std::shared_ptr<stream_ref>& stream,
                   std::array<uint32_t, 3> grid, uint32_t threads, void** params);

    int sm_count(int device);

    // ------------------------------------------------------------ operands --
    // A float32 operand read in place: device address of element 0 and its
    // strides (a strided view is not copied as long as its innermost axis is
    // contiguous). Ordered behind its producer on `stream`.
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

    // Sources of representative instantiations of every operator kernel, in
    // the "kernel <name> ..." format of describe_plan, for build checks.
    std::string operator_sources();
    void norm_rope_sources(std::vector<std::pair<std::string, std::string>>& out);

} // namespace porch::detail
