// Layer operators on device tensors: linear layers and their gradients,
// orthogonalised matrices and the optimiser step that takes them. Host interface
// of linear.cu and orthogonal.cu; arguments have been checked by the C entry
// points. Every call is asynchronous on `stream` and allocates nothing. `error` is
// a word of the host that a kernel sets when it gives up a wait.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace cpde::ops {

struct LinearCall {
    int32_t type, bias_type, activation;
    const void* x;
    int64_t x_stride;
    int64_t points, inputs, outputs;
    const void* weight;  // outputs rows of inputs
    int64_t weight_stride;
    const void* bias;
    const void* residual;
    int64_t residual_stride;
    void *y, *z;  // contiguous
    void* workspace;
};
size_t linear_workspace(const LinearCall& call);
void linear(const LinearCall& call, int* error, cudaStream_t stream);

struct LinearGradientCall {
    int32_t type, activation, weight_type, bias_type;  // the last two of dweight and dbias
    const void *grad, *z;
    int64_t grad_stride, z_stride;
    const void* x;
    int64_t x_stride;
    int64_t points, inputs, outputs;
    const void* weight;
    int64_t weight_stride;
    void *dx, *dweight, *dbias;  // contiguous; any may be null
    void* workspace;
};
size_t linear_gradient_workspace(const LinearGradientCall& call);
void linear_gradient(const LinearGradientCall& call, int* error, cudaStream_t stream);

// Matrices are contiguous. Coefficients are triples, `triples` of them: step k takes the k-th, or the last.
struct OrthogonalCall {
    int32_t type, momentum_type;
    int64_t matrices, rows, columns;
    int32_t steps, triples;
    const double* coefficients;
    double eps;
    const void* x;  // the matrices, or the gradient of an optimiser step
    void* out;      // the orthogonalised matrices, or the new weights
    // An optimiser step's:
    const void *weight, *momentum;
    void* new_momentum;
    double beta, keep, rate;  // new weights = keep * weight - rate * orthogonalised
    bool nesterov, step;
    void* workspace;
};
// Whether the singular values stay within what the parts can hold.
bool orthogonal_bounded(const OrthogonalCall& call);
size_t orthogonal_workspace(const OrthogonalCall& call);
void orthogonal(const OrthogonalCall& call, int* error, cudaStream_t stream);

// A wait that nothing ends and that gives up after some microseconds.
void give_up(int* error, cudaStream_t stream);

}  // namespace cpde::ops
