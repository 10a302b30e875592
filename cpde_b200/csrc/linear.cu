// Launches of linear layers and their gradients (layers.hpp).
#include "gemm_launch.hpp"
#include "kernels_linear.cuh"
#include "layers.hpp"

namespace cpde::ops {
namespace {

enum Type : int32_t { F32 = 0, BF16 = 1, F16 = 2 };

template <class T> struct Tag { using type = T; };
template <class F>
void with_type(int32_t type, F&& f) {
    if (type == F32) f(Tag<float>{});
    else if (type == BF16) f(Tag<__nv_bfloat16>{});
    else f(Tag<__half>{});
}

// Parts of a workspace, 256-byte aligned.
struct Room {
    char* base;
    size_t bytes = 0;
    template <class T> T* take(size_t count) {
        T* p = base ? reinterpret_cast<T*>(base + bytes) : nullptr;
        bytes += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

int64_t eights(int64_t n) { return (n + 7) / 8 * 8; }
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether TMA reads the array as it is: whole 16-byte units from row to row.
bool direct(int32_t type, const void* p, int64_t stride, int64_t rows) {
    return type != F32 && aligned(p, 16) && (rows == 1 || stride % 8 == 0);
}

int64_t row_chunks(int64_t rows, int64_t columns, int lanes) {
    const int64_t strips = (columns + 8 * lanes - 1) / (8 * lanes), high = 256 / lanes;
    // About eight blocks an SM, and four passes of a block's threads at least.
    return std::max<int64_t>(1, std::min<int64_t>({GEMM_SMS * 8 / strips, (rows + 4 * high - 1) / (4 * high), 1024}));
}
int row_lanes(int64_t columns) {
    int lanes = 1;
    while (lanes < 32 && lanes * 8 < columns) lanes *= 2;
    return lanes;
}

template <class T>
size_t parts_count(int64_t rows, int64_t columns) {
    return size_t(rows) * eights(columns) * Parts<T>::count;
}

// An array as an operand: as it is, or in parts of its own.
template <class T>
Operand staged(const T* x, int64_t stride, const T* z, int64_t z_stride, int32_t activation, int64_t rows, int64_t columns,
               typename Parts<T>::type* out, float* sums, cudaStream_t stream) {
    PartsCall<T> c = {};
    c.x = x, c.z = z, c.out = out, c.sums = sums;
    c.x_stride = stride, c.z_stride = z_stride, c.rows = rows;
    c.columns = int(columns), c.pitch = int(eights(columns)), c.activation = activation;
    c.lanes = row_lanes(columns);
    const int64_t chunks = row_chunks(rows, columns, c.lanes);
    c.chunk = (rows + chunks - 1) / chunks;
    constexpr int per = 16 / sizeof(T);
    c.whole = aligned(x, 16) && stride % per == 0 && (!z || (aligned(z, 16) && z_stride % per == 0));
    const dim3 grid(unsigned((columns + 8 * c.lanes - 1) / (8 * c.lanes)), unsigned(chunks));
    launch_early(k_parts<T>, grid, 256, 0, 1, stream, c);
    return {out, c.pitch, rows, columns, Parts<T>::count, rows * c.pitch, Parts<T>::count};
}

template <class T, bool A_ROWS, bool B_ROWS>
void product(const Operand& a, const Operand& b, int64_t m, int64_t n, int64_t k, const GemmPlan& plan,
             LinearEpilogue<T> epilogue, float* partial, int* error, cudaStream_t stream) {
    constexpr int P = Parts<T>::count;
    constexpr bool bf16 = !std::is_same_v<T, __half>;
    // Partial sums have whole rows, whatever the result's are.
    if (plan.splits > 1) epilogue.partial = partial, epilogue.whole = true;
    with_tile<P, A_ROWS, B_ROWS>(plan, [&](auto tile) {
        launch_gemm<decltype(tile)>(a, b, m, n, k, 1, bf16, false, plan, epilogue, error, stream);
    });
    if (plan.splits == 1) return;
    GemmShape s = {};
    s.m = int(m), s.n = int(n), s.splits = plan.splits;
    const int64_t threads = m * (epilogue.fours ? n / 4 : n);
    const dim3 grid(unsigned(std::min<int64_t>((threads + 255) / 256, GEMM_SMS * 8)));
    if (epilogue.fours) launch_early(k_join<T, 4>, grid, 256, 0, 1, stream, epilogue, s);
    else launch_early(k_join<T, 1>, grid, 256, 0, 1, stream, epilogue, s);
}

// Whether rows of `n` elements at these addresses take the wide accesses of the epilogue, and those of fours.
template <class T>
void set_widths(LinearEpilogue<T>& e, int64_t n) {
    auto all = [&](int count) {
        const int64_t own = count * sizeof(T), wide = count * 4;
        auto fits = [](const void* p, int64_t bytes) { return aligned(p, std::min<int64_t>(bytes, 32)); };
        return n % count == 0 && fits(e.y, e.y_wide ? wide : own) && fits(e.z, own) && fits(e.bias, e.bias_wide ? wide : own) &&
               fits(e.residual, own) && (!e.residual || e.residual_stride % count == 0);
    };
    e.whole = all(16), e.fours = all(4);
}

size_t partial_count(const GemmPlan& plan, int64_t m, int64_t n) {
    return plan.splits > 1 ? size_t(plan.splits) * m * ((n + 15) / 16 * 16) : 0;
}

template <class T>
size_t run_linear(const LinearCall& c, int* error, cudaStream_t stream, bool launch) {
    constexpr int P = Parts<T>::count;
    using O = typename Parts<T>::type;
    Room room = {launch ? static_cast<char*>(c.workspace) : nullptr};
    const bool x_direct = direct(c.type, c.x, c.x_stride, c.points), w_direct = direct(c.type, c.weight, c.weight_stride, c.outputs);
    const GemmPlan plan = gemm_plan<P>(c.points, c.outputs, c.inputs, 1, false, true);
    O* x_parts = x_direct ? nullptr : room.take<O>(parts_count<T>(c.points, c.inputs));
    O* w_parts = w_direct ? nullptr : room.take<O>(parts_count<T>(c.outputs, c.inputs));
    float* partial = room.take<float>(partial_count(plan, c.points, c.outputs));
    if (!launch) return room.bytes;
    const T *x = static_cast<const T*>(c.x), *w = static_cast<const T*>(c.weight);
    const Operand a = x_direct ? Operand{x, c.x_stride, c.points, c.inputs, 1, 0, 1}
                               : staged<T>(x, c.x_stride, nullptr, 0, 1, c.points, c.inputs, x_parts, nullptr, stream);
    const Operand b = w_direct ? Operand{w, c.weight_stride, c.outputs, c.inputs, 1, 0, 1}
                               : staged<T>(w, c.weight_stride, nullptr, 0, 1, c.outputs, c.inputs, w_parts, nullptr, stream);
    LinearEpilogue<T> e = {};
    e.bias = c.bias, e.bias_wide = c.bias_type == F32;
    e.residual = static_cast<const T*>(c.residual), e.residual_stride = c.residual_stride;
    e.z = static_cast<T*>(c.z), e.y = c.y, e.y_wide = c.type == F32;
    e.activation = c.activation;
    set_widths(e, c.outputs);
    product<T, false, false>(a, b, c.points, c.outputs, c.inputs, plan, e, partial, error, stream);
    return room.bytes;
}

template <class T>
size_t run_gradient(const LinearGradientCall& c, int* error, cudaStream_t stream, bool launch) {
    constexpr int P = Parts<T>::count;
    using O = typename Parts<T>::type;
    Room room = {launch ? static_cast<char*>(c.workspace) : nullptr};
    const bool sloped = c.activation != 1;
    const bool dz_direct = !sloped && direct(c.type, c.grad, c.grad_stride, c.points);
    const bool x_direct = !c.dweight || direct(c.type, c.x, c.x_stride, c.points);
    const bool w_direct = !c.dx || direct(c.type, c.weight, c.weight_stride, c.outputs);
    const bool products = c.dx || c.dweight;
    const GemmPlan dx_plan = gemm_plan<P>(c.points, c.inputs, c.outputs, 1, false, true);
    const GemmPlan dw_plan = gemm_plan<P>(c.outputs, c.inputs, c.points, 1, false, true);
    O* dz_parts = dz_direct || !products ? nullptr : room.take<O>(parts_count<T>(c.points, c.outputs));
    O* x_parts = x_direct ? nullptr : room.take<O>(parts_count<T>(c.points, c.inputs));
    O* w_parts = w_direct ? nullptr : room.take<O>(parts_count<T>(c.outputs, c.inputs));
    const int64_t chunks = row_chunks(c.points, c.outputs, row_lanes(c.outputs));
    float* sums = c.dbias ? room.take<float>(chunks * c.outputs) : nullptr;
    float* partial = room.take<float>(std::max(c.dx ? partial_count(dx_plan, c.points, c.inputs) : 0,
                                               c.dweight ? partial_count(dw_plan, c.outputs, c.inputs) : 0));
    if (!launch) return room.bytes;
    const T *grad = static_cast<const T*>(c.grad), *z = sloped ? static_cast<const T*>(c.z) : nullptr;
    const T *x = static_cast<const T*>(c.x), *w = static_cast<const T*>(c.weight);
    Operand dz = {grad, c.grad_stride, c.points, c.outputs, 1, 0, 1};
    if (dz_parts || c.dbias) {
        const Operand made = staged<T>(grad, c.grad_stride, z, c.z_stride, c.activation, c.points, c.outputs, dz_parts, sums, stream);
        if (dz_parts) dz = made;
    }
    if (c.dbias) {
        const dim3 grid(unsigned((c.outputs + 31) / 32));
        if (c.bias_type == F32)
            launch_early(k_column_sums<float>, grid, 256, 0, 1, stream, sums, int32_t(chunks), int32_t(c.outputs),
                         static_cast<float*>(c.dbias));
        else
            launch_early(k_column_sums<T>, grid, 256, 0, 1, stream, sums, int32_t(chunks), int32_t(c.outputs),
                         static_cast<T*>(c.dbias));
    }
    LinearEpilogue<T> e = {};
    e.activation = 1;
    if (c.dx) {
        const Operand b = w_direct ? Operand{w, c.weight_stride, c.outputs, c.inputs, 1, 0, 1}
                                   : staged<T>(w, c.weight_stride, nullptr, 0, 1, c.outputs, c.inputs, w_parts, nullptr, stream);
        e.y = c.dx, e.y_wide = c.type == F32;
        set_widths(e, c.inputs);
        product<T, false, true>(dz, b, c.points, c.inputs, c.outputs, dx_plan, e, partial, error, stream);
    }
    if (c.dweight) {
        const Operand b = x_direct ? Operand{x, c.x_stride, c.points, c.inputs, 1, 0, 1}
                                   : staged<T>(x, c.x_stride, nullptr, 0, 1, c.points, c.inputs, x_parts, nullptr, stream);
        e.y = c.dweight, e.y_wide = c.weight_type == F32;
        set_widths(e, c.inputs);
        product<T, true, true>(dz, b, c.outputs, c.inputs, c.points, dw_plan, e, partial, error, stream);
    }
    return room.bytes;
}

}  // namespace

size_t linear_workspace(const LinearCall& call) {
    size_t bytes = 0;
    with_type(call.type, [&](auto t) { bytes = run_linear<typename decltype(t)::type>(call, nullptr, nullptr, false); });
    return bytes;
}
void linear(const LinearCall& call, int* error, cudaStream_t stream) {
    with_type(call.type, [&](auto t) { run_linear<typename decltype(t)::type>(call, error, stream, true); });
}
size_t linear_gradient_workspace(const LinearGradientCall& call) {
    size_t bytes = 0;
    with_type(call.type, [&](auto t) { bytes = run_gradient<typename decltype(t)::type>(call, nullptr, nullptr, false); });
    return bytes;
}
void linear_gradient(const LinearGradientCall& call, int* error, cudaStream_t stream) {
    with_type(call.type, [&](auto t) { run_gradient<typename decltype(t)::type>(call, error, stream, true); });
}

}  // namespace cpde::ops
