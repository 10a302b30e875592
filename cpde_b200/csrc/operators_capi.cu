// C entry points of the device-tensor operators: argument checks, then the
// launches of operators.cu.
#include "operators.hpp"

#include <algorithm>

namespace {

using cpde::require;

constexpr int64_t kMostIndexed = (int64_t(1) << 31) - 2;
constexpr int64_t kMostChannels = int64_t(1) << 20;

size_t type_bytes(int32_t type) {
    require(type == CPDE_F32 || type == CPDE_BF16 || type == CPDE_F16, "element type must be 0 (f32), 1 (bf16) or 2 (f16)");
    return type == CPDE_F32 ? 4 : 2;
}

void check_array(const void* p, size_t element, const char* name) {
    require(p, std::string(name) + " is a null device pointer");
    require(reinterpret_cast<uintptr_t>(p) % element == 0, std::string(name) + " is not aligned to its element type");
}

void check_ids(int32_t id_type, const void* ids, int64_t tokens) {
    require(id_type == CPDE_I32 || id_type == CPDE_I64, "id type must be 0 (int32) or 1 (int64)");
    if (tokens) check_array(ids, id_type == CPDE_I64 ? 8 : 4, "ids");
}

void check_embedding(int64_t tokens, int64_t rows, int64_t channels) {
    require(rows > 0 && rows <= kMostIndexed && tokens >= 0 && tokens <= kMostIndexed,
            "rows must be positive, tokens not negative, and both below 2^31 - 1");
    require(channels > 0 && channels <= kMostChannels, "channels must be between 1 and 2^20");
}

void check_dropout(double rate) { require(rate >= 0 && rate <= 1, "the dropout rate must be between 0 and 1"); }

void check_norm(int64_t instances, int64_t points, int64_t channels, int64_t groups) {
    require(instances >= 0 && points >= 0 && points <= kMostIndexed,
            "instances and points must not be negative, points below 2^31 - 1");
    require(channels > 0 && channels <= kMostChannels, "channels must be between 1 and 2^20");
    require(groups > 0 && channels % groups == 0, "the group count must divide the channels");
    require(instances <= (int64_t(1) << 20), "instances must be at most 2^20");
}

void check_norm_call(const cpde::ops::NormCall& c) {
    check_norm(c.instances, c.points, c.channels, c.groups);
    const size_t element = type_bytes(c.type);
    require(c.parameter_type == CPDE_F32 || c.parameter_type == c.type,
            "weight and bias must be f32 or of the array's type");
    require(c.activation >= 0 && c.activation <= 3, "activation must be 0 (sigmoid), 1 (linear), 2 (tanh) or 3 (SiLU)");
    check_dropout(c.rate);
    const size_t parameter = type_bytes(c.parameter_type);
    if (c.weight) check_array(c.weight, parameter, "weight");
    if (c.bias) check_array(c.bias, parameter, "bias");
    if (c.lengths) check_array(c.lengths, 4, "lengths");
    if (!c.instances) return;
    check_array(c.mean, 4, "mean");
    check_array(c.rstd, 4, "rstd");
    if (!c.points) return;
    check_array(c.x, element, "x");
    check_array(c.out, element, "the output");
    require(c.x_point >= c.channels || c.points == 1, "x's point stride must be at least the channels");
    require(c.x_instance >= 0, "x's instance stride must not be negative");
}

void check_workspace(const void* workspace, size_t bytes, size_t needed) {
    if (!needed) return;
    require(bytes >= needed, "the workspace must have " + std::to_string(needed) + " bytes");
    check_array(workspace, 256, "workspace");
}

// As guard(), and the caller's current device stays what it was: these calls mix
// with those of a program that has a device of its own. A kernel that gave up a wait
// in an earlier call is reported here: such a program may make no other call.
template <class F>
int guard_operator(cpde_engine* h, F&& f) {
    int before = 0;
    const bool known = h && h->engine && cudaGetDevice(&before) == cudaSuccess;
    const int status = guard(h, [&] {
        h->engine->check_operator_errors();
        f();
    });
    if (known && before != h->engine->device) cudaSetDevice(before);
    return status;
}

// A workspace size for a caller.
template <class F>
int query(size_t* bytes, F&& f) {
    if (!bytes) return CPDE_REJECTED;
    try {
        *bytes = f();
        return CPDE_OK;
    } catch (...) {
        return CPDE_REJECTED;
    }
}

size_t norm_workspace(int64_t instances, int64_t points, int64_t channels, int64_t groups, bool gradient) {
    return instances && points ? cpde::ops::group_norm_workspace(instances, points, channels, groups, gradient) : 0;
}

cudaStream_t stream_of(cpde_engine* h, void* stream) {
    return stream ? static_cast<cudaStream_t>(stream) : h->engine->stream;
}

}  // namespace

extern "C" {

int cpde_embedding(cpde_engine* h, int32_t table_type, const void* table, int64_t table_stride, int64_t rows,
                   int64_t channels, int32_t id_type, const void* ids, int64_t tokens, float scale, int32_t out_type,
                   void* out, void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(table_type), out_element = type_bytes(out_type);
        require(out_type == table_type || table_type == CPDE_F32, "the output's type must be the table's, or the table f32");
        check_embedding(tokens, rows, channels);
        check_ids(id_type, ids, tokens);
        require(table_stride >= channels || rows == 1, "the table's stride must be at least the channels");
        if (!tokens) return;
        check_array(table, element, "table");
        check_array(out, out_element, "out");
        cpde::ops::embedding({table_type, out_type, id_type, table, table_stride, ids, out, tokens, rows, channels, scale,
                              nullptr},
                             stream_of(h, stream));
    });
}

int cpde_embedding_gradient_workspace(int64_t tokens, int64_t rows, int64_t channels, size_t* bytes) {
    return query(bytes, [&] {
        check_embedding(tokens, rows, channels);
        return cpde::ops::embedding_gradient_workspace(tokens, rows, channels);
    });
}

int cpde_embedding_gradient(cpde_engine* h, int32_t grad_type, const void* grad, int64_t grad_stride,
                            int32_t id_type, const void* ids, int64_t tokens, int64_t rows, int64_t channels,
                            float scale, int32_t out_type, void* out, void* workspace, size_t workspace_bytes,
                            void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(grad_type), out_element = type_bytes(out_type);
        require(out_type == grad_type || out_type == CPDE_F32, "the output's type must be the gradient's or f32");
        check_embedding(tokens, rows, channels);
        check_ids(id_type, ids, tokens);
        check_array(out, out_element, "out");
        if (tokens) {
            check_array(grad, element, "grad");
            require(grad_stride >= channels || tokens == 1, "the gradient's stride must be at least the channels");
            check_workspace(workspace, workspace_bytes, cpde::ops::embedding_gradient_workspace(tokens, rows, channels));
        }
        cpde::ops::embedding_gradient({grad_type, out_type, id_type, grad, grad_stride, ids, out, tokens, rows, channels,
                                       scale, workspace},
                                      h->engine->device, stream_of(h, stream));
    });
}

int cpde_dropout(cpde_engine* h, int32_t type, const void* x, int64_t x_stride, const void* residual,
                 int64_t residual_stride, int64_t rows, int64_t columns, double rate, uint64_t seed, uint64_t offset,
                 void* y, void* stream) {
    return guard_operator(h, [&] {
        const size_t element = type_bytes(type);
        check_dropout(rate);
        require(rows >= 0 && columns >= 0, "rows and columns must not be negative");
        if (!rows || !columns) return;
        require(columns <= (int64_t(1) << 41) / rows, "at most 2^41 elements");
        check_array(x, element, "x");
        check_array(y, element, "y");
        if (residual) check_array(residual, element, "residual");
        require(rows == 1 || (x_stride >= columns && (!residual || residual_stride >= columns)),
                "strides must be at least the columns");
        cpde::ops::dropout({type, x, x_stride, residual, residual_stride, y, rows, columns, rate, seed, offset},
                           stream_of(h, stream));
    });
}

int cpde_group_norm_workspace(int64_t instances, int64_t points, int64_t channels, int64_t groups, size_t* bytes) {
    return query(bytes, [&] {
        check_norm(instances, points, channels, groups);
        return std::max(norm_workspace(instances, points, channels, groups, false),
                        norm_workspace(instances, points, channels, groups, true));
    });
}

int cpde_group_norm_forward_workspace(int64_t instances, int64_t points, int64_t channels, int64_t groups, size_t* bytes) {
    return query(bytes, [&] {
        check_norm(instances, points, channels, groups);
        return norm_workspace(instances, points, channels, groups, false);
    });
}

int cpde_group_norm(cpde_engine* h, int32_t type, const void* x, int64_t x_point_stride,
                    int64_t x_instance_stride, int64_t instances, int64_t points, int64_t channels, int64_t groups,
                    int32_t parameter_type, const void* weight, const void* bias, double eps, int32_t activation,
                    const int32_t* lengths, double rate, uint64_t seed, uint64_t offset, void* y, float* mean,
                    float* rstd, void* workspace, size_t workspace_bytes, void* stream) {
    return guard_operator(h, [&] {
        cpde::ops::NormCall c = {};
        c.type = type, c.parameter_type = parameter_type, c.activation = activation;
        c.x = x, c.x_point = x_point_stride, c.x_instance = x_instance_stride;
        c.instances = instances, c.points = points, c.channels = channels, c.groups = groups;
        c.weight = weight, c.bias = bias, c.lengths = lengths;
        c.eps = eps, c.rate = rate, c.seed = seed, c.offset = offset;
        c.out = y, c.mean = mean, c.rstd = rstd, c.workspace = workspace;
        check_norm_call(c);
        require(float(eps) > 0, "eps must be positive, also in FP32");
        check_workspace(workspace, workspace_bytes, norm_workspace(instances, points, channels, groups, false));
        cpde::ops::group_norm(c, h->engine->device, stream_of(h, stream));
    });
}

int cpde_group_norm_gradient(cpde_engine* h, int32_t type, const void* grad, int64_t grad_point_stride,
                             int64_t grad_instance_stride, const void* x, int64_t x_point_stride,
                             int64_t x_instance_stride, const float* mean, const float* rstd, int64_t instances,
                             int64_t points, int64_t channels, int64_t groups, int32_t parameter_type,
                             const void* weight, const void* bias, int32_t activation, const int32_t* lengths,
                             double rate, uint64_t seed, uint64_t offset, void* dx, void* dweight, void* dbias,
                             void* workspace, size_t workspace_bytes, void* stream) {
    return guard_operator(h, [&] {
        cpde::ops::NormCall c = {};
        c.type = type, c.parameter_type = parameter_type, c.activation = activation;
        c.x = x, c.x_point = x_point_stride, c.x_instance = x_instance_stride;
        c.grad = grad, c.grad_point = grad_point_stride, c.grad_instance = grad_instance_stride;
        c.instances = instances, c.points = points, c.channels = channels, c.groups = groups;
        c.weight = weight, c.bias = bias, c.lengths = lengths;
        c.rate = rate, c.seed = seed, c.offset = offset;
        c.out = dx, c.mean = const_cast<float*>(mean), c.rstd = const_cast<float*>(rstd);
        c.dweight = dweight, c.dbias = dbias, c.workspace = workspace;
        check_norm_call(c);
        const size_t parameter = type_bytes(parameter_type);
        if (dweight) check_array(dweight, parameter, "dweight");
        if (dbias) check_array(dbias, parameter, "dbias");
        if (instances && points) {
            check_array(grad, type_bytes(type), "grad");
            require(grad_point_stride >= channels || points == 1, "the gradient's point stride must be at least the channels");
            require(grad_instance_stride >= 0, "the gradient's instance stride must not be negative");
            check_workspace(workspace, workspace_bytes, norm_workspace(instances, points, channels, groups, true));
        }
        cpde::ops::group_norm_gradient(c, h->engine->device, stream_of(h, stream));
    });
}

}  // extern "C"
