// Launches of linear layers and their gradients (layers.hpp).
#include "gemm_launch.hpp"
#include "kernels_few.cuh"
#include "layers.hpp"

namespace cpde::ops {
namespace {

template <class F>
void with_type(int32_t type, F&& f) {
    if (type == F32) f(Tag<float>{});
    else if (type == BF16) f(Tag<__nv_bfloat16>{});
    else f(Tag<__half>{});
}

// Layers of at most so many points (or outputs) may take the kernel that reads the other side once.
constexpr int64_t FEW_POINTS = 8;

int64_t eights(int64_t n) { return (n + 7) / 8 * 8; }

// Whether TMA reads the array as it is: whole 16-byte units from row to row.
bool direct(int32_t type, const void* p, int64_t stride, int64_t rows) {
    return type != F32 && aligned(p, 16) && (rows == 1 || stride % 8 == 0);
}

int64_t row_chunks(int64_t rows, int64_t columns, int lanes) {
    const int64_t strips = (columns + 8 * lanes - 1) / (8 * lanes), high = 256 / lanes;
    // About eight blocks an SM, and four passes of a block's threads at least.
    return std::max<int64_t>(1, std::min<int64_t>({GEMM_SMS * 8 / strips, (rows + 4 * high - 1) / (4 * high), 1024}));
}

template <class T>
size_t parts_count(int64_t rows, int64_t columns) {
    return size_t(rows) * eights(columns) * Parts<T>::count;
}

// Adds an array to those that are made into parts, and gives the operand that it becomes;
// `out` may be null where the column sums alone are wanted.
template <class T>
Operand staged(PartsCalls<T>& calls, const T* x, int64_t stride, const T* z, int64_t z_stride, int32_t activation, int64_t rows,
               int64_t columns, typename Parts<T>::type* out, float* sums) {
    PartsCall<T>& c = calls.call[calls.count++];
    c.x = x, c.z = z, c.out = out, c.sums = sums;
    c.x_stride = stride, c.z_stride = z_stride, c.rows = rows;
    c.columns = int(columns), c.pitch = int(eights(columns)), c.activation = activation;
    c.lanes = row_lanes(columns);
    const int64_t chunks = row_chunks(rows, columns, c.lanes);
    c.chunk = (rows + chunks - 1) / chunks;
    c.strips = int((columns + 8 * c.lanes - 1) / (8 * c.lanes)), c.blocks = int(c.strips * chunks);
    constexpr int per = 16 / sizeof(T);
    c.whole = aligned(x, 16) && stride % per == 0 && (!z || (aligned(z, 16) && z_stride % per == 0));
    return {out, c.pitch, rows, columns, Parts<T>::count, rows * c.pitch, Parts<T>::count};
}
template <class T>
void launch_parts(const PartsCalls<T>& calls, cudaStream_t stream) {
    int64_t blocks = 0;
    for (int i = 0; i < calls.count; ++i) blocks += calls.call[i].blocks;
    if (blocks) launch_early(k_parts<T>, dim3(unsigned(blocks)), 256, 0, 1, stream, calls);
}

template <class T>
Source<T> source(const T* p, int64_t stride, int64_t rows, int64_t columns) {
    int width = 8;
    while (width > 1 && !(aligned(p, width * sizeof(T)) && (rows == 1 || stride % width == 0))) width /= 2;
    return {p, stride, rows, int32_t(columns), width};
}

// How a product is computed: on operands that TMA reads, `a_made` and `b_made` being made
// for it, or gathered from the arrays in one launch.
struct Route {
    GemmPlan plan;
    bool gather;
};
// An operand: whether TMA reads it, and what there is to make into parts otherwise.
struct Side {
    bool there;
    int64_t elements;
};
template <class T>
Route route(int64_t m, int64_t n, int64_t k, const Side& a, const Side& b) {
    constexpr int P = Parts<T>::count;
    Route r = {gemm_plan<P>(m, n, k, 1, false, true), false};
    if (a.there && b.there) return r;
    // Parts: read and written at about 2000 bytes a clock, and a launch.
    double made = r.plan.clocks;
    for (const Side* s : {&a, &b})
        if (!s->there) made += LAUNCH_CLOCKS + double(s->elements) * (sizeof(T) + 2 * P) / 2000;
    // Gathered, where B's parts stay in shared memory: 65,536 points of 128 inputs and outputs
    // in FP32 take 40 us instead of 51 with parts. At 64 outputs half of its tile is empty:
    // 25 instead of 20.
    if constexpr (P > 1) {
        const bool resident = n <= 128 && P * ((k + GEMM_SLAB - 1) / GEMM_SLAB) <= GemmTile<1, 128, P, false, false, true>::HELD;
        if (!resident || n <= 64) return r;
        GemmPlan gathered = {};
        consider(gathered, 1, 128, 4500, m, n, k, 1, false, false);
        if (gathered.clocks < made) r = {gathered, true};
    }
    return r;
}

size_t partial_count(const GemmPlan& plan, int64_t m, int64_t n) {
    return plan.splits > 1 ? size_t(plan.splits) * m * ((n + 15) / 16 * 16) : 0;
}

template <class T>
void join(const GemmPlan& plan, int64_t m, int64_t n, const LinearEpilogue<T>& epilogue, cudaStream_t stream) {
    if (plan.splits == 1) return;
    GemmShape s = {};
    s.m = int(m), s.n = int(n), s.splits = plan.splits;
    const int64_t threads = m * (epilogue.fours ? n / 4 : n);
    // Few results of many splits: a warp's threads share the splits of one.
    const int share = plan.splits >= 16 && threads <= GEMM_SMS * 256 ? 8 : 1;
    const dim3 grid(unsigned(std::min<int64_t>((threads * share + 255) / 256, GEMM_SMS * 8)));
    if (epilogue.fours) launch_early(k_join<T, 4>, grid, 256, 0, 1, stream, epilogue, s, share);
    else launch_early(k_join<T, 1>, grid, 256, 0, 1, stream, epilogue, s, share);
}

// Partial sums have whole rows, whatever the result's are.
template <class T>
LinearEpilogue<T> split_epilogue(const GemmPlan& plan, LinearEpilogue<T> epilogue, float* partial) {
    if (plan.splits > 1) epilogue.partial = partial, epilogue.whole = true;
    return epilogue;
}

template <class T, bool A_ROWS, bool B_ROWS>
void product(const Operand& a, const Operand& b, int64_t m, int64_t n, int64_t k, const GemmPlan& plan,
             const LinearEpilogue<T>& epilogue, float* partial, int* error, cudaStream_t stream) {
    constexpr int P = Parts<T>::count;
    constexpr bool bf16 = !std::is_same_v<T, __half>;
    const LinearEpilogue<T> e = split_epilogue(plan, epilogue, partial);
    with_tile<P, A_ROWS, B_ROWS>(plan, [&](auto tile) {
        launch_gemm<decltype(tile)>(a, b, m, n, k, 1, bf16, false, plan, e, error, stream);
    });
    join(plan, m, n, e, stream);
}

template <class C, class T>
void launch_gather(const Source<T>& a, const Source<T>& b, int64_t m, int64_t n, int64_t k, const GemmPlan& plan,
                   const LinearEpilogue<T>& epilogue, int* error, cudaStream_t stream) {
    constexpr bool bf16 = !std::is_same_v<T, __half>;
    GemmShape s = gemm_shape(m, n, k, 1, C::BM, C::BN, false, plan);
    s.instruction = mma_instruction(C::BM, C::BN, C::A_ROWS, C::B_ROWS, bf16);
    static std::atomic<uint64_t> ready{0};
    allow_shared(k_gather<C, T, LinearEpilogue<T>>, C::SHARED, ready);
    const int64_t items = int64_t(s.tiles) * s.splits;
    launch_early(k_gather<C, T, LinearEpilogue<T>>, dim3(unsigned(std::min<int64_t>(items, GEMM_SMS))), GATHER_THREADS<C>, C::SHARED, 1,
                 stream, a, b, s, epilogue, error);
}
template <class T, bool B_ROWS>
void gathered_product(const Source<T>& a, const Source<T>& b, int64_t m, int64_t n, int64_t k, const Route& r,
                      const LinearEpilogue<T>& epilogue, int* error, cudaStream_t stream) {
    if constexpr (Parts<T>::count > 1)
        launch_gather<GemmTile<1, 128, Parts<T>::count, false, B_ROWS, true>>(a, b, m, n, k, r.plan, epilogue, error, stream);
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

// Products on the FP32 units in blocks of 32 x 32, and the microseconds that they take: an SM has
// one block at a time, which goes through its slabs one after the other. Against them stand the
// launches of the tensor cores' tiles, which for layers of this size take about as long each
// whatever it is. Measured, blocks against tiles: 1000 x 64 -> 64 FP32 5.0 and 10.2, 600 x 128 ->
// 128 6.3 and 10.9, 100 x 512 -> 64 13.4 and 12.8; bf16 5.3 and 5.5, 6.7 and 5.9, 14.3 and 6.7 in
// whole 16 bytes, 5.2 and 8.9, 6.7 and 9.1, 14.3 and 10.0 where x and W are copied; 1440 x 64 ->
// 1440 bf16 58 and 8.3. Gradients of 300 x 104 -> 80 with SiLU and bias FP32 13.4 and 29.4, bf16
// 13.0 and 20.4, of 1000 x 64 -> 64 34.6 and 26.1, 30.2 and 20.6.
struct SmallWork {
    int64_t blocks = 0, slabs = 0;
    void add(int64_t m, int64_t n, int64_t k) {
        blocks += ((m + SMALL_TILE - 1) / SMALL_TILE) * ((n + SMALL_TILE - 1) / SMALL_TILE);
        slabs = std::max(slabs, (k + SMALL_SLAB - 1) / SMALL_SLAB);
    }
    double time(double slab) const { return 1.1 + double((blocks + GEMM_SMS - 1) / GEMM_SMS) * (2.8 + slab * slabs); }
};
template <class T>
SmallProduct<T> small_call(const SmallOperand<T>& a, const SmallOperand<T>& b, int64_t m, int64_t n, int64_t k,
                           const LinearEpilogue<T>& e) {
    const int64_t tiles_n = (n + SMALL_TILE - 1) / SMALL_TILE;
    return {a, b, e, nullptr, false, int32_t(m), int32_t(n), int32_t(tiles_n), k, int32_t((m + SMALL_TILE - 1) / SMALL_TILE * tiles_n)};
}
template <class T>
void launch_small(const SmallProduct<T>& first, const SmallProduct<T>& second, cudaStream_t stream) {
    launch_early(k_small_products<T>, dim3(unsigned(first.tiles + second.tiles)), 32 * SMALL_WARPS, 0, 1, stream, first, second);
}

template <class T, bool TURNED>
void launch_few(const Source<T>& x, const Source<T>& w, const LinearEpilogue<T>& e, cudaStream_t stream) {
    GemmShape s = {};
    s.m = int(TURNED ? w.rows : x.rows), s.n = int(TURNED ? x.rows : w.rows);
    auto go = [&](auto points) {
        constexpr int POINTS = decltype(points)::value;
        const int64_t each = FEW_THREADS / 32 * FEW_OUTPUTS<POINTS>;
        launch_early(k_few_points<T, POINTS, TURNED>, dim3(unsigned((w.rows + each - 1) / each)), FEW_THREADS, 0, 1, stream, x, w, e, s);
    };
    if (x.rows == 1) go(std::integral_constant<int, 1>{});
    else if (x.rows == 2) go(std::integral_constant<int, 2>{});
    else if (x.rows <= 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
}

template <class T>
size_t run_linear(const LinearCall& c, int* error, cudaStream_t stream, bool launch) {
    using O = typename Parts<T>::type;
    Room room = {launch ? static_cast<char*>(c.workspace) : nullptr};
    const T *x = static_cast<const T*>(c.x), *w = static_cast<const T*>(c.weight);
    const Source<T> xs = source(x, c.x_stride, c.points, c.inputs), ws = source(w, c.weight_stride, c.outputs, c.inputs);
    LinearEpilogue<T> e = {};
    e.bias = c.bias, e.bias_wide = c.bias_type == F32;
    e.residual = static_cast<const T*>(c.residual), e.residual_stride = c.residual_stride;
    e.z = static_cast<T*>(c.z), e.y = c.y, e.y_wide = c.type == F32;
    e.activation = c.activation;
    set_widths(e, c.outputs);
    // A warp's way through a row takes the same time up to 64 inputs a sum that it holds, so
    // rows shorter than that are for the tensor cores if there are many: a million points of
    // 16 inputs and 8 outputs take 171 us there in FP32 and 924 here, 20,000 of 2048 and 4
    // take 126 and 38, 65,536 of 512 and 8 take 99 both; 16-bit x (21 and 24 us) is never
    // turned.
    const auto long_rows = [&](int64_t sums) {
        int64_t held = 2;
        while (held < sums) held *= 2;
        return c.inputs >= 64 * held;
    };
    const bool few = c.points <= FEW_POINTS && (c.outputs <= 16384 || long_rows(c.points));
    const bool turned = c.type == F32 && c.outputs <= FEW_POINTS && long_rows(c.outputs);
    const bool x_direct = direct(c.type, x, c.x_stride, c.points), w_direct = direct(c.type, w, c.weight_stride, c.outputs);
    SmallWork work;
    work.add(c.points, c.outputs, c.inputs);
    const bool small = work.time(1.3) <= (sizeof(T) == 4 ? 11.0 : x_direct && w_direct ? 5.6 : 8.8);
    if (few || turned || small) {
        if (!launch) return 0;
        if (few) {
            launch_few<T, false>(xs, ws, e, stream);
        } else if (turned) {
            if constexpr (sizeof(T) == 4) launch_few<T, true>(ws, xs, e, stream);
        } else {
            launch_small(small_call<T>({x, nullptr, c.x_stride, 1}, {w, nullptr, c.weight_stride, 1}, c.points, c.outputs, c.inputs, e),
                         {}, stream);
        }
        return 0;
    }
    const Route r = route<T>(c.points, c.outputs, c.inputs, {x_direct, c.points * c.inputs},
                             {w_direct, c.outputs * c.inputs});
    O* x_parts = x_direct || r.gather ? nullptr : room.take<O>(parts_count<T>(c.points, c.inputs));
    O* w_parts = w_direct || r.gather ? nullptr : room.take<O>(parts_count<T>(c.outputs, c.inputs));
    float* partial = room.take<float>(partial_count(r.plan, c.points, c.outputs));
    if (!launch) return room.bytes;
    if (r.gather) {
        gathered_product<T, false>(xs, ws, c.points, c.outputs, c.inputs, r, e, error, stream);
        return room.bytes;
    }
    PartsCalls<T> parts = {};
    const Operand a = x_direct ? Operand{x, c.x_stride, c.points, c.inputs, 1, 0, 1}
                               : staged<T>(parts, x, c.x_stride, nullptr, 0, 1, c.points, c.inputs, x_parts, nullptr);
    const Operand b = w_direct ? Operand{w, c.weight_stride, c.outputs, c.inputs, 1, 0, 1}
                               : staged<T>(parts, w, c.weight_stride, nullptr, 0, 1, c.outputs, c.inputs, w_parts, nullptr);
    launch_parts(parts, stream);
    product<T, false, false>(a, b, c.points, c.outputs, c.inputs, r.plan, e, partial, error, stream);
    return room.bytes;
}

template <class T>
size_t run_gradient(const LinearGradientCall& c, int* error, cudaStream_t stream, bool launch) {
    if (!c.dx && !c.dweight && !c.dbias) return 0;
    using O = typename Parts<T>::type;
    Room room = {launch ? static_cast<char*>(c.workspace) : nullptr};
    const bool sloped = c.activation != 1;
    const T *grad = static_cast<const T*>(c.grad), *z = sloped ? static_cast<const T*>(c.z) : nullptr;
    const T *x = static_cast<const T*>(c.x), *w = static_cast<const T*>(c.weight);
    const bool dz_direct = !sloped && direct(c.type, grad, c.grad_stride, c.points);
    const bool x_direct = direct(c.type, x, c.x_stride, c.points), w_direct = direct(c.type, w, c.weight_stride, c.outputs);
    SmallWork work;
    if (c.dx) work.add(c.points, c.inputs, c.outputs);
    if (c.dweight || c.dbias) work.add(c.outputs, c.dweight ? c.inputs : 1, c.points);
    // Parts, the bias' sums (a pass of their own if nothing becomes parts) and the products.
    const bool parts_made = !dz_direct || (c.dweight && !x_direct) || (c.dx && !w_direct);
    const double tiles = (parts_made ? sloped ? 8.0 : 4.0 : 0.0) + (c.dbias ? parts_made ? 2.0 : 4.5 : 0.0) +
                         ((c.dx != nullptr) + (c.dweight != nullptr)) * (sizeof(T) == 4 ? 7.5 : 5.6);
    if (work.time(sloped ? 1.9 : 1.2) <= tiles) {
        if (!launch) return 0;
        LinearEpilogue<T> e = {};
        e.activation = 1;
        const int64_t zs = c.z_stride;
        SmallProduct<T> dx = {}, dw = {};
        if (c.dx) {
            e.y = c.dx, e.y_wide = c.type == F32;
            set_widths(e, c.inputs);
            dx = small_call<T>({grad, z, c.grad_stride, 1, zs, 1, c.activation}, {w, nullptr, 1, c.weight_stride}, c.points, c.inputs,
                               c.outputs, e);
        }
        if (c.dweight || c.dbias) {
            // dbias alone is the rows' sums of a product without columns.
            e.y = c.dweight, e.y_wide = c.weight_type == F32;
            set_widths(e, c.inputs);
            dw = small_call<T>({grad, z, 1, c.grad_stride, 1, zs, c.activation}, {x, nullptr, 1, c.x_stride}, c.outputs,
                               c.dweight ? c.inputs : 1, c.points, e);
            if (!c.dweight) dw.n = 0;
            dw.sums = c.dbias, dw.sums_wide = c.bias_type == F32;
        }
        launch_small(dx, dw, stream);
        return 0;
    }
    // dz is made in the type's parts where the activation has a slope; otherwise it is
    // grad, which is made into parts only if a product is not gathered.
    const Source<T> gs = source(grad, c.grad_stride, c.points, c.outputs), ws = source(w, c.weight_stride, c.outputs, c.inputs);
    Route dx = {};
    if (c.dx && !sloped) dx = route<T>(c.points, c.inputs, c.outputs, {dz_direct, c.points * c.outputs}, {w_direct, c.outputs * c.inputs});
    else dx.plan = gemm_plan<Parts<T>::count>(c.points, c.inputs, c.outputs, 1, false, true);
    // An FP32 gradient of 16-bit weights: the sum goes over dz and over what rounding it to the
    // type has left, so that it is good to 16 bits and more a term. For gradients of the type
    // their own rounding is as large as dz's, and the second half of the sum would take as long
    // as the first: 32,768 points of 2048 x 2048 bf16 500 us, 720 with it.
    const bool rest = sizeof(T) == 2 && sloped && c.dweight && c.weight_type == F32;
    const int64_t dw_terms = rest ? 2 * ((c.points + GEMM_SLAB - 1) / GEMM_SLAB) * GEMM_SLAB : c.points;
    const GemmPlan dw_plan = gemm_plan<Parts<T>::count>(c.outputs, c.inputs, dw_terms, 1, false, true);
    const bool made = (c.dx && !dx.gather) || c.dweight;
    O* dz_parts = dz_direct || !made ? nullptr : room.take<O>(parts_count<T>(c.points, c.outputs) * (rest ? 2 : 1));
    O* x_parts = x_direct || !c.dweight ? nullptr : room.take<O>(parts_count<T>(c.points, c.inputs));
    O* w_parts = w_direct || !c.dx || dx.gather ? nullptr : room.take<O>(parts_count<T>(c.outputs, c.inputs));
    const int64_t chunks = row_chunks(c.points, c.outputs, row_lanes(c.outputs));
    float* sums = c.dbias ? room.take<float>(chunks * c.outputs) : nullptr;
    float* partial = room.take<float>(std::max(c.dx ? partial_count(dx.plan, c.points, c.inputs) : 0,
                                               c.dweight ? partial_count(dw_plan, c.outputs, c.inputs) : 0));
    if (!launch) return room.bytes;
    Operand dz = {grad, c.grad_stride, c.points, c.outputs, 1, 0, 1}, xo = {x, c.x_stride, c.points, c.inputs, 1, 0, 1},
            wo = {w, c.weight_stride, c.outputs, c.inputs, 1, 0, 1};
    PartsCalls<T> parts = {};
    if (dz_parts || c.dbias) {
        const Operand o = staged<T>(parts, grad, c.grad_stride, z, c.z_stride, c.activation, c.points, c.outputs, dz_parts, sums);
        if (dz_parts) dz = o;
        if (rest) parts.call[parts.count - 1].rest = true, dz.planes = 2;
    }
    if (w_parts) wo = staged<T>(parts, w, c.weight_stride, nullptr, 0, 1, c.outputs, c.inputs, w_parts, nullptr);
    if (x_parts) xo = staged<T>(parts, x, c.x_stride, nullptr, 0, 1, c.points, c.inputs, x_parts, nullptr);
    launch_parts(parts, stream);
    if (c.dbias) {
        const dim3 grid(unsigned((c.outputs + 31) / 32));
        if (c.bias_type == F32)
            launch_early(k_column_sums<float>, grid, 1024, 0, 1, stream, sums, int32_t(chunks), int32_t(c.outputs),
                         static_cast<float*>(c.dbias));
        else
            launch_early(k_column_sums<T>, grid, 1024, 0, 1, stream, sums, int32_t(chunks), int32_t(c.outputs),
                         static_cast<T*>(c.dbias));
    }
    LinearEpilogue<T> e = {};
    e.activation = 1;
    if (c.dx) {
        e.y = c.dx, e.y_wide = c.type == F32;
        set_widths(e, c.inputs);
        if (dx.gather) gathered_product<T, true>(gs, ws, c.points, c.inputs, c.outputs, dx, e, error, stream);
        else product<T, false, true>(dz, wo, c.points, c.inputs, c.outputs, dx.plan, e, partial, error, stream);
    }
    if (c.dweight) {
        e.y = c.dweight, e.y_wide = c.weight_type == F32;
        set_widths(e, c.inputs);
        product<T, true, true>(dz, xo, c.outputs, c.inputs, dw_terms, dw_plan, e, partial, error, stream);
    }
    return room.bytes;
}

__global__ void k_give_up(int* error) {
    __shared__ uint64_t never;
    tc::mbar_init(&never, 1);
    tc::fence_barrier_init();
    if (!tc::mbar_wait(&never, 0, 10000)) gemm::report(error);
}

}  // namespace

void give_up(int* error, cudaStream_t stream) {
    k_give_up<<<1, 1, 0, stream>>>(error);
    CPDE_LAUNCHED();
}
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
