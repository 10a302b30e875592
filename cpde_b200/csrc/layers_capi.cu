// C entry points of the layer operators: argument checks, then the launches of
// linear.cu and orthogonal.cu. Included behind operators_capi.cu, whose checks it shares.
#include <cmath>

#include "layers.hpp"

namespace {

// Rows of the last tile count as 31-bit numbers too.
constexpr int64_t kMostPoints = (int64_t(1) << 31) - 512;

void check_linear(int64_t points, int64_t inputs, int64_t outputs) {
    require(points >= 0 && points <= kMostPoints, "points must not be negative, and at most 2^31 - 512");
    require(inputs > 0 && inputs <= kMostChannels && outputs > 0 && outputs <= kMostChannels,
            "inputs and outputs must be between 1 and 2^20");
}

void check_activation(int32_t activation) {
    require(activation >= 0 && activation <= 3, "activation must be 0 (sigmoid), 1 (linear), 2 (tanh) or 3 (SiLU)");
}

void check_rows(const void* p, size_t element, int64_t stride, int64_t rows, int64_t columns, const char* name) {
    check_array(p, element, name);
    require(stride >= columns || rows == 1, std::string(name) + "'s row stride must be at least its columns");
}

void check_parameter(int32_t parameter, int32_t type, const char* message) {
    require(parameter == CPDE_F32 || parameter == type, message);
}

cpde::ops::LinearCall linear_call(int32_t type, const void* x, int64_t x_stride, int64_t points, int64_t inputs, int64_t outputs,
                                  const void* weight, int64_t weight_stride) {
    cpde::ops::LinearCall c = {};
    type_bytes(type);
    check_linear(points, inputs, outputs);
    c.type = type, c.x = x, c.x_stride = x_stride;
    c.points = points, c.inputs = inputs, c.outputs = outputs;
    c.weight = weight, c.weight_stride = weight_stride;
    return c;
}

// Bits of the gradients that are wanted.
constexpr int32_t kWantInput = 1, kWantWeight = 2, kWantBias = 4, kWeightOfType = 8;

cpde::ops::LinearGradientCall gradient_call(int32_t type, const void* grad, int64_t grad_stride, int32_t activation, const void* x,
                                            int64_t x_stride, int64_t points, int64_t inputs, int64_t outputs,
                                            const void* weight, int64_t weight_stride) {
    cpde::ops::LinearGradientCall c = {};
    type_bytes(type);
    check_linear(points, inputs, outputs);
    check_activation(activation);
    c.type = type, c.activation = activation;
    c.grad = grad, c.grad_stride = grad_stride, c.x = x, c.x_stride = x_stride;
    c.points = points, c.inputs = inputs, c.outputs = outputs;
    c.weight = weight, c.weight_stride = weight_stride;
    return c;
}

void check_matrices(int64_t matrices, int64_t rows, int64_t columns) {
    require(matrices >= 0 && matrices <= 65535, "there must be at most 65535 matrices");
    require(rows > 0 && rows <= kMostChannels && columns > 0 && columns <= kMostChannels,
            "rows and columns must be between 1 and 2^20");
}

void check_steps(cpde::ops::OrthogonalCall& c, int32_t steps, const double* coefficients, int32_t triples, double eps) {
    require(steps >= 1 && steps <= 64, "steps must be between 1 and 64");
    require(coefficients && triples >= 1 && triples <= steps, "coefficients must be triples, one at least and at most one a step");
    for (int32_t i = 0; i < 3 * triples; ++i) require(std::isfinite(coefficients[i]), "coefficients must be finite");
    require(eps >= 1e-30 && eps < 1e30, "eps must be between 1e-30 and 1e30");
    c.steps = steps, c.coefficients = coefficients, c.triples = triples, c.eps = eps;
    require(cpde::ops::orthogonal_bounded(c), "with these coefficients a singular value may pass 1024");
}

}  // namespace

extern "C" {

int cpde_operator_check(cpde_engine* h) { return guard_operator(h, [] {}); }

int cpde_operator_give_up(cpde_engine* h, void* stream) {
    return guard_operator(h, [&] { cpde::ops::give_up(h->engine->operator_error_device, stream_of(h, stream)); });
}

int cpde_linear_workspace(int32_t type, const void* x, int64_t x_stride, int64_t points, int64_t inputs, int64_t outputs,
                          const void* weight, int64_t weight_stride, size_t* bytes) {
    return query(bytes, [&] {
        const auto c = linear_call(type, x, x_stride, points, inputs, outputs, weight, weight_stride);
        return points ? cpde::ops::linear_workspace(c) : 0;
    });
}

int cpde_linear(cpde_engine* h, int32_t type, const void* x, int64_t x_stride, int64_t points, int64_t inputs, int64_t outputs,
                const void* weight, int64_t weight_stride, int32_t bias_type, const void* bias, int32_t activation,
                const void* residual, int64_t residual_stride, void* y, void* z, void* workspace, size_t workspace_bytes,
                void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(type);
        auto c = linear_call(type, x, x_stride, points, inputs, outputs, weight, weight_stride);
        check_activation(activation);
        check_parameter(bias_type, type, "bias must be f32 or of the array's type");
        if (!points) return;
        check_rows(x, element, x_stride, points, inputs, "x");
        check_rows(weight, element, weight_stride, outputs, inputs, "weight");
        if (bias) check_array(bias, type_bytes(bias_type), "bias");
        if (residual) check_rows(residual, element, residual_stride, points, outputs, "residual");
        check_array(y, element, "y");
        if (z) check_array(z, element, "z");
        c.bias_type = bias_type, c.bias = bias, c.activation = activation;
        c.residual = residual, c.residual_stride = residual_stride;
        c.y = y, c.z = z, c.workspace = workspace;
        check_workspace(workspace, workspace_bytes, cpde::ops::linear_workspace(c));
        cpde::ops::linear(c, h->engine->operator_error_device, stream_of(h, stream));
    });
}

int cpde_linear_gradient_workspace(int32_t type, const void* grad, int64_t grad_stride, int32_t activation, const void* x,
                                   int64_t x_stride, int64_t points, int64_t inputs, int64_t outputs, const void* weight,
                                   int64_t weight_stride, int32_t want, size_t* bytes) {
    return query(bytes, [&] {
        auto c = gradient_call(type, grad, grad_stride, activation, x, x_stride, points, inputs, outputs, weight, weight_stride);
        static char wanted;
        c.dx = want & kWantInput ? &wanted : nullptr;
        c.dweight = want & kWantWeight ? &wanted : nullptr;
        c.dbias = want & kWantBias ? &wanted : nullptr;
        if (!points) return size_t(0);
        c.weight_type = type;
        size_t bytes = cpde::ops::linear_gradient_workspace(c);
        if (want & kWeightOfType) return bytes;
        c.weight_type = CPDE_F32;
        return std::max(bytes, cpde::ops::linear_gradient_workspace(c));
    });
}

int cpde_linear_gradient(cpde_engine* h, int32_t type, const void* grad, int64_t grad_stride, const void* z, int64_t z_stride,
                         int32_t activation, const void* x, int64_t x_stride, int64_t points, int64_t inputs, int64_t outputs,
                         const void* weight, int64_t weight_stride, void* dx, int32_t weight_type, void* dweight,
                         int32_t bias_type, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(type);
        auto c = gradient_call(type, grad, grad_stride, activation, x, x_stride, points, inputs, outputs, weight, weight_stride);
        check_parameter(weight_type, type, "dweight must be f32 or of the array's type");
        check_parameter(bias_type, type, "dbias must be f32 or of the array's type");
        if (dweight) check_array(dweight, type_bytes(weight_type), "dweight");
        if (dbias) check_array(dbias, type_bytes(bias_type), "dbias");
        const cudaStream_t s = stream_of(h, stream);
        if (!points) {  // sums of nothing
            if (dweight) CPDE_CUDA(cudaMemsetAsync(dweight, 0, size_t(outputs) * inputs * type_bytes(weight_type), s));
            if (dbias) CPDE_CUDA(cudaMemsetAsync(dbias, 0, size_t(outputs) * type_bytes(bias_type), s));
            return;
        }
        check_rows(grad, element, grad_stride, points, outputs, "grad");
        if (activation != 1) check_rows(z, element, z_stride, points, outputs, "z");
        if (dweight) check_rows(x, element, x_stride, points, inputs, "x");
        if (dx) check_rows(weight, element, weight_stride, outputs, inputs, "weight"), check_array(dx, element, "dx");
        c.z = z, c.z_stride = z_stride, c.weight_type = weight_type, c.bias_type = bias_type;
        c.dx = dx, c.dweight = dweight, c.dbias = dbias, c.workspace = workspace;
        check_workspace(workspace, workspace_bytes, cpde::ops::linear_gradient_workspace(c));
        cpde::ops::linear_gradient(c, h->engine->operator_error_device, s);
    });
}

int cpde_orthogonalize_workspace(int32_t type, int64_t matrices, int64_t rows, int64_t columns, size_t* bytes) {
    return query(bytes, [&] {
        type_bytes(type);
        check_matrices(matrices, rows, columns);
        cpde::ops::OrthogonalCall c = {};
        c.type = type, c.matrices = matrices, c.rows = rows, c.columns = columns;
        return matrices ? cpde::ops::orthogonal_workspace(c) : 0;
    });
}

int cpde_orthogonalize(cpde_engine* h, int32_t type, const void* x, int64_t matrices, int64_t rows, int64_t columns, int32_t steps,
                       const double* coefficients, int32_t triples, double eps, void* out, void* workspace,
                       size_t workspace_bytes, void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(type);
        check_matrices(matrices, rows, columns);
        cpde::ops::OrthogonalCall c = {};
        check_steps(c, steps, coefficients, triples, eps);
        if (!matrices) return;
        check_array(x, element, "x");
        check_array(out, element, "out");
        c.type = type, c.matrices = matrices, c.rows = rows, c.columns = columns;
        c.x = x, c.out = out, c.workspace = workspace;
        check_workspace(workspace, workspace_bytes, cpde::ops::orthogonal_workspace(c));
        cpde::ops::orthogonal(c, h->engine->operator_error_device, stream_of(h, stream));
    });
}

int cpde_muon_workspace(int32_t type, int64_t rows, int64_t columns, size_t* bytes) {
    return query(bytes, [&] {
        type_bytes(type);
        check_matrices(1, rows, columns);
        cpde::ops::OrthogonalCall c = {};
        c.type = type, c.matrices = 1, c.rows = rows, c.columns = columns, c.step = true;
        return cpde::ops::orthogonal_workspace(c);
    });
}

int cpde_muon(cpde_engine* h, int32_t type, const void* weight, const void* grad, int32_t momentum_type, const void* momentum,
              int64_t rows, int64_t columns, double rate, double beta, int32_t nesterov, double decay, double scale, int32_t steps,
              const double* coefficients, int32_t triples, double eps, void* new_weight, void* new_momentum, void* workspace,
              size_t workspace_bytes, void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(type);
        check_matrices(1, rows, columns);
        check_parameter(momentum_type, type, "momentum must be f32 or of the weight's type");
        require(beta >= 0 && beta < 1, "beta must be at least 0 and below 1");
        require(std::isfinite(rate) && std::isfinite(decay) && std::isfinite(scale), "rate, decay and scale must be finite");
        cpde::ops::OrthogonalCall c = {};
        check_steps(c, steps, coefficients, triples, eps);
        for (const void* p : {weight, grad, static_cast<const void*>(new_weight)}) check_array(p, element, "weight, grad or the new weight");
        check_array(momentum, type_bytes(momentum_type), "momentum");
        check_array(new_momentum, type_bytes(momentum_type), "the new momentum");
        c.type = type, c.momentum_type = momentum_type, c.matrices = 1, c.rows = rows, c.columns = columns;
        c.x = grad, c.weight = weight, c.out = new_weight, c.momentum = momentum, c.new_momentum = new_momentum;
        c.beta = beta, c.nesterov = nesterov != 0, c.keep = 1 - rate * decay, c.rate = rate * scale, c.step = true;
        c.workspace = workspace;
        check_workspace(workspace, workspace_bytes, cpde::ops::orthogonal_workspace(c));
        cpde::ops::orthogonal(c, h->engine->operator_error_device, stream_of(h, stream));
    });
}

}  // extern "C"
