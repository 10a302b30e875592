// Device-tensor operators: embedding lookup and its gradient, dropout, group
// norm with an activation and its gradient. Host interface of operators.cu;
// arguments have been checked by the C entry points. Every call is asynchronous
// on `stream` and allocates nothing.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace cpde::ops {

struct EmbeddingCall {
    int32_t in_type, out_type, id_type;
    const void* in;       // table (rows x channels), or gradient (tokens x channels)
    int64_t in_stride;    // elements between rows of `in`
    const void* ids;
    void* out;            // contiguous
    int64_t tokens, rows, channels;
    float scale;
    void* workspace;
};
void embedding(const EmbeddingCall& call, cudaStream_t stream);
size_t embedding_gradient_workspace(int64_t tokens, int64_t rows, int64_t channels);
void embedding_gradient(const EmbeddingCall& call, int device, cudaStream_t stream);

struct DropoutCall {
    int32_t type;
    const void* x;
    int64_t x_stride;
    const void* residual;
    int64_t residual_stride;
    void* y;  // contiguous
    int64_t rows, columns;
    double rate;
    uint64_t seed, offset;
};
void dropout(const DropoutCall& call, cudaStream_t stream);

struct NormCall {
    int32_t type, parameter_type, activation;
    const void* x;
    int64_t x_point, x_instance;
    const void* grad;  // gradient only
    int64_t grad_point, grad_instance;
    int64_t instances, points, channels, groups;
    const void *weight, *bias;
    const int32_t* lengths;
    double eps, rate;
    uint64_t seed, offset;
    void* out;  // y or dx, contiguous
    float *mean, *rstd;
    void *dweight, *dbias;
    void* workspace;
};
size_t group_norm_workspace(int64_t instances, int64_t points, int64_t channels, int64_t groups, bool gradient);
void group_norm(const NormCall& call, int device, cudaStream_t stream);
void group_norm_gradient(const NormCall& call, int device, cudaStream_t stream);

}  // namespace cpde::ops
