// Launches of orthogonalised matrices and the optimiser step (layers.hpp).
#include <cmath>
#include <vector>

#include "gemm_launch.hpp"
#include "kernels_orthogonal_small.cuh"
#include "layers.hpp"

namespace cpde::ops {
namespace {

struct Step {
    double a, b, c;
    int x, gram, poly;  // exponents of what the step holds: X, A and Q
};

double largest(double a, double b, double c, double to) {
    // |a s + b s^3 + c s^5| on [0, to]: at its end or where the derivative is zero.
    auto at = [&](double t) { return std::fabs(std::sqrt(t) * (a + t * (b + t * c))); };
    double most = at(to * to);
    const double d = 9 * b * b - 20 * a * c;
    double roots[2] = {-1, -1};
    if (c != 0 && d >= 0) roots[0] = (-3 * b + std::sqrt(d)) / (10 * c), roots[1] = (-3 * b - std::sqrt(d)) / (10 * c);
    else if (c == 0 && b != 0) roots[0] = -a / (3 * b);
    for (double t : roots)
        if (t > 0 && t < to * to) most = std::max(most, at(t));
    return most;
}
double largest_poly(double b, double c, double to) {
    auto at = [&](double t) { return std::fabs(t * (b + t * c)); };
    double most = at(to);
    const double t = c != 0 ? -b / (2 * c) : -1;
    if (t > 0 && t < to) most = std::max(most, at(t));
    return most;
}
// Largest power of two by which a matrix without an entry above `bound` stays within FP16.
int exponent(double bound) { return std::min(30, int(std::floor(std::log2(32768.0 / std::max(bound, 1e-6))))); }

// The steps' coefficients and exponents; false where the singular values pass 1024.
bool plan_steps(const OrthogonalCall& c, std::vector<Step>& steps) {
    double bound = 1.0 + 1e-5;
    for (int k = 0; k < c.steps; ++k) {
        const double* v = c.coefficients + 3 * std::min(k, c.triples - 1);
        Step s = {v[0], v[1], v[2], exponent(bound), exponent(bound * bound), 0};
        const double poly = largest_poly(v[1], v[2], bound * bound) * 1.01;
        s.poly = exponent(poly);
        bound = largest(v[0], v[1], v[2], bound) * 1.01;  // and a margin for the steps' own errors
        if (!(bound < 1024) || !(poly < 16384)) return false;
        steps.push_back(s);
    }
    return true;
}

// Whether one CTA holds a matrix.
bool small(const OrthogonalCall& c) {
    return std::min(c.rows, c.columns) <= SMALL_SIDE && std::max(c.rows, c.columns) <= SMALL_LENGTH;
}

template <class T, class M>
void run_small(const OrthogonalCall& c, int* error, cudaStream_t stream) {
    std::vector<Step> steps;
    plan_steps(c, steps);
    SmallCall<T, M> s = {};
    s.x = static_cast<const T*>(c.x);
    s.out = static_cast<T*>(c.out);
    if (c.step) {
        s.momentum = static_cast<const M*>(c.momentum), s.new_momentum = static_cast<M*>(c.new_momentum);
        s.weight = static_cast<const T*>(c.weight);
        s.beta = float(c.beta), s.rest = float(1 - c.beta), s.keep = float(c.keep), s.rate = float(c.rate);
        s.nesterov = c.nesterov;
    }
    s.rows = int(c.rows), s.columns = int(c.columns), s.steps = c.steps;
    s.whole = c.columns % 8 == 0;
    for (const void* p : {c.x, static_cast<const void*>(c.out), s.weight ? c.weight : nullptr, s.momentum ? c.momentum : nullptr,
                          static_cast<const void*>(s.new_momentum)})
        s.whole = s.whole && aligned(p, 16);
    s.scale = std::ldexp(1.0f, steps[0].x), s.eps = c.eps;
    for (int k = 0; k < c.steps; ++k) {
        const Step& v = steps[k];
        const int next = k + 1 < c.steps ? steps[k + 1].x : 0;
        s.step[k] = {std::ldexp(1.0f, v.gram - 2 * v.x), float(std::ldexp(v.b, v.poly - v.gram)),
                     float(std::ldexp(v.c, v.poly - 2 * v.gram)), float(std::ldexp(v.a, next - v.x)),
                     float(std::ldexp(1.0, next - v.x - v.poly))};
    }
    const int64_t side = std::min(c.rows, c.columns), length = std::max(c.rows, c.columns);
    const size_t shared = 1024 + ((length + 63) / 64 + (side + 63) / 64) * 2 * SMALL_BLOCK;
    static std::atomic<uint64_t> ready{0};
    allow_shared(k_orthogonal_small<T, M>, 1024 + 12 * SMALL_BLOCK, ready);
    launch_early(k_orthogonal_small<T, M>, dim3(unsigned(c.matrices)), SMALL_THREADS, shared, 1, stream, s, error);
}

template <int P, class T, class M>
size_t run(const OrthogonalCall& c, int* error, cudaStream_t stream, bool launch) {
    if (small(c)) {
        if constexpr (P == 2)
            if (launch) run_small<T, M>(c, error, stream);
        return 0;
    }
    const int64_t m = c.rows, n = c.columns, side = std::min(m, n), batch = c.matrices;
    const bool tall = m > n;
    const int64_t pitch = (n + 15) / 16 * 16, gram_pitch = (side + 15) / 16 * 16;
    const int lanes = row_lanes(n), high = 256 / lanes;
    const int blocks = int(std::max<int64_t>(
        1, std::min<int64_t>({(m + high - 1) / high, (GEMM_SMS * 8 + batch - 1) / batch, 1024})));
    Room room = {launch ? static_cast<char*>(c.workspace) : nullptr};
    double* sums = room.take<double>(batch * blocks);
    float* update = c.step ? room.take<float>(m * n) : nullptr;
    __half* x[2];
    for (auto& p : x) p = room.take<__half>(2 * batch * m * pitch);
    __half* gram = room.take<__half>(P * batch * side * gram_pitch);
    __half* poly = room.take<__half>(P * batch * side * gram_pitch);
    if (!launch) return room.bytes;

    std::vector<Step> steps;
    plan_steps(c, steps);
    const float first = std::ldexp(1.0f, steps[0].x);
    const int64_t plane = m * pitch, gram_plane = side * gram_pitch;
    UpdateCall<T, M> u = {};
    u.x = static_cast<const T*>(c.x);
    if (c.step) u.momentum = static_cast<const M*>(c.momentum), u.new_momentum = static_cast<M*>(c.new_momentum);
    u.update = update, u.sums = sums;
    u.rows = m, u.columns = int(n), u.lanes = lanes, u.blocks = blocks;
    u.beta = float(c.beta), u.rest = float(1 - c.beta), u.nesterov = c.nesterov;
    u.whole = n % 8 == 0 && aligned(c.x, 16) && (!c.step || (aligned(c.momentum, 16) && aligned(c.new_momentum, 16)));
    const dim3 grid{unsigned(blocks), unsigned(batch)};
    launch_early(k_update_norm<T, M>, grid, 256, 0, 1, stream, u);
    if (c.step)
        launch_early(k_normalise<float>, grid, 256, 0, 1, stream, update, sums, x[0], m, pitch, plane, int32_t(n), lanes, blocks,
                     first, c.eps, n % 8 == 0);
    else
        launch_early(k_normalise<T>, grid, 256, 0, 1, stream, u.x, sums, x[0], m, pitch, plane, int32_t(n), lanes, blocks, first,
                     c.eps, u.whole);

    const GemmPlan gram_plan = gemm_plan<P>(side, side, std::max(m, n), batch, true, false);
    const GemmPlan square_plan = gemm_plan<P>(side, side, side, batch, true, false);
    const GemmPlan step_plan = gemm_plan<P>(m, n, side, batch, false, false);
    const Operand g = {gram, gram_pitch, side, side, P * batch, gram_plane, P};
    const Operand q = {poly, gram_pitch, side, side, P * batch, gram_plane, P};
    for (int k = 0; k < c.steps; ++k) {
        const Step& s = steps[k];
        const Operand in = {x[k & 1], pitch, m, n, 2 * batch, plane, 2};
        OrthogonalEpilogue<true, 0, P, T> to_gram = {};
        to_gram.out = gram, to_gram.pitch = gram_pitch, to_gram.plane = gram_plane, to_gram.out_planes = P;
        to_gram.whole = true;
        to_gram.scale_d = std::ldexp(1.0f, s.gram - 2 * s.x);
        if (tall)
            with_tile<P, true, true>(gram_plan, [&](auto tile) {
                launch_gemm<decltype(tile)>(in, in, side, side, m, batch, false, true, gram_plan, to_gram, error, stream);
            });
        else
            with_tile<P, false, false>(gram_plan, [&](auto tile) {
                launch_gemm<decltype(tile)>(in, in, side, side, n, batch, false, true, gram_plan, to_gram, error, stream);
            });
        OrthogonalEpilogue<true, P, P, T> to_poly = {};
        to_poly.in = gram, to_poly.out = poly, to_poly.pitch = gram_pitch, to_poly.plane = gram_plane;
        to_poly.whole = true;
        to_poly.in_planes = to_poly.out_planes = P;
        to_poly.scale_in = float(std::ldexp(s.b, s.poly - s.gram)), to_poly.scale_d = float(std::ldexp(s.c, s.poly - 2 * s.gram));
        with_tile<P, false, false>(square_plan, [&](auto tile) {
            launch_gemm<decltype(tile)>(g, g, side, side, side, batch, false, true, square_plan, to_poly, error, stream);
        });
        auto step = [&](auto epilogue, int next) {
            epilogue.in = x[k & 1], epilogue.pitch = pitch, epilogue.plane = plane;
            epilogue.in_planes = epilogue.out_planes = 2;
            epilogue.scale_in = float(std::ldexp(s.a, next - s.x)), epilogue.scale_d = float(std::ldexp(1.0, next - s.x - s.poly));
            if (tall)
                with_tile<P, false, false>(step_plan, [&](auto tile) {
                    launch_gemm<decltype(tile)>(in, q, m, n, side, batch, false, false, step_plan, epilogue, error, stream);
                });
            else
                with_tile<P, false, true>(step_plan, [&](auto tile) {
                    launch_gemm<decltype(tile)>(q, in, m, n, side, batch, false, false, step_plan, epilogue, error, stream);
                });
        };
        if (k + 1 < c.steps) {
            OrthogonalEpilogue<false, 2, 2, T> e = {};
            e.out = x[(k + 1) & 1], e.whole = true;
            step(e, steps[k + 1].x);
        } else {
            OrthogonalEpilogue<false, 2, 0, T> e = {};
            e.final = static_cast<T*>(c.out);
            if (c.step) e.weight = static_cast<const T*>(c.weight), e.keep = float(c.keep), e.rate = float(c.rate);
            e.whole = n % 16 == 0 && aligned(c.out, 32) && aligned(e.weight, 32);
            step(e, 0);
        }
    }
    return room.bytes;
}

// Products of both parts for FP32; for FP16 matrices, whose own rounding is as small as the
// steps' error with one part (not for FP16 weights, of which a step is a small fraction);
// and where the smaller side is up to 256: there the errors do not average out, and the
// products take no time.
size_t run_types(const OrthogonalCall& c, int* error, cudaStream_t stream, bool launch) {
    auto with = [&](auto element, auto momentum, bool both) {
        using T = typename decltype(element)::type;
        using M = typename decltype(momentum)::type;
        if constexpr (sizeof(T) == 2)
            if (!both) return run<1, T, M>(c, error, stream, launch);
        return run<2, T, M>(c, error, stream, launch);
    };
    const bool wide = c.step && c.momentum_type == F32;
    const bool both = std::min(c.rows, c.columns) <= 256 || (c.type == F16 && !c.step);
    if (c.type == F32) return with(Tag<float>{}, Tag<float>{}, true);
    if (c.type == BF16) return wide ? with(Tag<__nv_bfloat16>{}, Tag<float>{}, both) : with(Tag<__nv_bfloat16>{}, Tag<__nv_bfloat16>{}, both);
    return wide ? with(Tag<__half>{}, Tag<float>{}, both) : with(Tag<__half>{}, Tag<__half>{}, both);
}

}  // namespace

bool orthogonal_bounded(const OrthogonalCall& call) {
    std::vector<Step> steps;
    return plan_steps(call, steps);
}
size_t orthogonal_workspace(const OrthogonalCall& call) { return run_types(call, nullptr, nullptr, false); }
void orthogonal(const OrthogonalCall& call, int* error, cudaStream_t stream) { run_types(call, error, stream, true); }

}  // namespace cpde::ops
