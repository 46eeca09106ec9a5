// nt_norm.hip — the operators between a transformer's matrix products: layer
// norm, dropout, and the residual edge that joins them (dropout of a branch,
// added to the residual stream, then the norm of the sum), each with its
// backward pass.
//
// With t a row of W elements (the input, or dropout(x) + residual):
//   mean = sum t / W, var = sum (t - mean)^2 / W, rstd = 1 / sqrt(var + eps)
//   y    = (t - mean) rstd w + b
// and with h = (t - mean) rstd, g = dy w:
//   dt   = rstd (g - sum g / W - h sum(g h) / W)   (+ the gradient that the sum gets from elsewhere)
//   dw   = sum over rows of dy h,   db = sum over rows of dy.
//
// Every sum and statistic is float32; values are rounded once, when stored.
// The sums over rows run in two stages of fixed order, so gradients do not
// change from run to run.
#include <hip/hip_runtime.h>

#include <initializer_list>

#include "nt_internal.hpp"
#include "nt_philox.hpp"
#include "nt_pool.hpp"

namespace nt {

// What the edge does to its input before the norm.
enum Edge { kNone = 0, kAdd = 1, kDropAdd = 2 };

struct NormForward {
    const void *x, *residual, *weight, *bias;
    void *total, *y;
    float *mean, *rstd;         // may be null (both)
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    float eps;
    Mask mask;
};

struct NormBackward {
    const void *dy, *dtotal, *t, *weight;
    const float *mean, *rstd;
    void *dx, *dresidual;       // the edge writes both, the norm dx alone
    float *partials;            // [groups][2][width]
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    Mask mask;
};

__device__ __forceinline__ float load_param(const void *base, int32_t dtype, uint64_t i, float absent) {
    if (base == nullptr) return absent;
    switch (dtype) {
        case NT_F32: return reinterpret_cast<const float *>(base)[i];
        case NT_F16: return f16_to_f32(reinterpret_cast<const uint16_t *>(base)[i]);
        default: return bf16_to_f32(reinterpret_cast<const uint16_t *>(base)[i]);
    }
}

__device__ __forceinline__ float drop_one(float v, uint64_t i, const Mask &m) {
    const PhiloxWords words = philox(i >> 3, m.offset, m.seed);
    return philox_half(words, (int)(i & 7)) >= m.threshold ? v * m.factor : 0.0f;
}

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Sum over the workgroup, the same value on every lane; `shared` holds one
// float per wave.
__device__ __forceinline__ float block_sum_f32(float v, float *shared) {
    v = wave_sum_f32(v);
    __syncthreads();                                    // the last reader of `shared` is done
    if ((threadIdx.x & 63u) == 0u) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    float total = 0.0f;
    for (uint32_t k = 0; k < blockDim.x / 64u; ++k) total += shared[k];
    return total;
}

// ---- rows of any width: a workgroup per row, the row read once per pass ---------------------
template <class T, int EDGE>
__device__ __forceinline__ float row_value(const NormForward &a, uint64_t i) {
    float v = load1<T>(reinterpret_cast<const typename T::raw *>(a.x), i);
    if constexpr (EDGE == kDropAdd) v = drop_one(v, i, a.mask);
    if constexpr (EDGE != kNone) v += load1<T>(reinterpret_cast<const typename T::raw *>(a.residual), i);
    return v;
}

template <class T, int EDGE>
__global__ __launch_bounds__(kBlock) void norm_rows_kernel(NormForward a) {
    __shared__ float shared[kBlock / 64];
    const float width = (float)a.width;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width;
        float sum = 0.0f;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float v = row_value<T, EDGE>(a, base + c);
            if constexpr (EDGE != kNone) store1<T>(reinterpret_cast<typename T::raw *>(a.total), base + c, v);
            sum += v;
        }
        const float mean = block_sum_f32(sum, shared) / width;
        float squares = 0.0f;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float d = row_value<T, EDGE>(a, base + c) - mean;
            squares = __builtin_fmaf(d, d, squares);
        }
        const float rstd = 1.0f / __builtin_sqrtf(block_sum_f32(squares, shared) / width + a.eps);
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float h = (row_value<T, EDGE>(a, base + c) - mean) * rstd;
            store1<T>(reinterpret_cast<typename T::raw *>(a.y), base + c,
                      __builtin_fmaf(h, load_param(a.weight, a.weight_dtype, c, 1.0f),
                                     load_param(a.bias, a.weight_dtype, c, 0.0f)));
        }
        if (a.mean != nullptr && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <class T, int EDGE>
__global__ __launch_bounds__(kBlock) void norm_rows_backward_kernel(NormBackward a) {
    __shared__ float shared[kBlock / 64];
    const auto *dy = reinterpret_cast<const typename T::raw *>(a.dy);
    const auto *t = reinterpret_cast<const typename T::raw *>(a.t);
    const auto *dtotal = reinterpret_cast<const typename T::raw *>(a.dtotal);
    const float width = (float)a.width;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float level = 0.0f, along = 0.0f;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float g = load1<T>(dy, base + c) * load_param(a.weight, a.weight_dtype, c, 1.0f);
            level += g;
            along = __builtin_fmaf(g, (load1<T>(t, base + c) - mean) * rstd, along);
        }
        level = block_sum_f32(level, shared) / width;
        along = block_sum_f32(along, shared) / width;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float g = load1<T>(dy, base + c) * load_param(a.weight, a.weight_dtype, c, 1.0f);
            const float h = (load1<T>(t, base + c) - mean) * rstd;
            float d = rstd * (g - level - h * along);
            if constexpr (EDGE != kNone) {
                if (dtotal != nullptr) d += load1<T>(dtotal, base + c);
                store1<T>(reinterpret_cast<typename T::raw *>(a.dresidual), base + c, d);
                if constexpr (EDGE == kDropAdd) d = drop_one(d, base + c, a.mask);
            }
            store1<T>(reinterpret_cast<typename T::raw *>(a.dx), base + c, d);
        }
    }
}

// Column sums of dy h and dy over the rows that this workgroup's y index
// strides over, one column per lane.
template <class T>
__global__ __launch_bounds__(kBlock) void norm_columns_kernel(NormBackward a) {
    const uint32_t c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.width) return;
    const auto *dy = reinterpret_cast<const typename T::raw *>(a.dy);
    const auto *t = reinterpret_cast<const typename T::raw *>(a.t);
    float dw = 0.0f, db = 0.0f;
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = load1<T>(dy, row * a.width + c);
        dw = __builtin_fmaf(g, (load1<T>(t, row * a.width + c) - a.mean[row]) * a.rstd[row], dw);
        db += g;
    }
    float *out = a.partials + (uint64_t)blockIdx.y * 2u * a.width;
    out[c] = dw;
    out[a.width + c] = db;
}

// dw and db from the partial sums, rounded to the weight's dtype.
template <class T>
__global__ __launch_bounds__(kBlock) void norm_finalize_kernel(const float *partials, uint32_t groups, uint32_t width,
                                                               typename T::raw *dw, typename T::raw *db) {
    const uint64_t c = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= 2u * (uint64_t)width) return;
    typename T::raw *out = c < width ? dw : db;
    if (out == nullptr) return;
    float sum = 0.0f;
    for (uint32_t k = 0; k < groups; ++k) sum += partials[(uint64_t)k * 2u * width + c];
    store1<T>(out, c < width ? c : c - width, sum);
}

// ---- dropout over a flat tensor ----------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const typename T::raw *x, typename T::raw *y, uint64_t n,
                                                         Mask mask) {
    const uint64_t groups = (n + 7) >> 3;
    for (uint64_t g = (uint64_t)blockIdx.x * kBlock + threadIdx.x; g < groups; g += (uint64_t)gridDim.x * kBlock) {
        const PhiloxWords words = philox(g, mask.offset, mask.seed);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint64_t i = (g << 3) + k;
            if (i < n) {
                const float v = load1<T>(x, i) * mask.factor;
                store1<T>(y, i, philox_half(words, k) >= mask.threshold ? v : 0.0f);
            }
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------
constexpr uint32_t kColumnGroups = 256;                 // row groups of the column sums
constexpr uint64_t kMaxPartials = 256ull << 20;         // bytes of their workspace
constexpr uint64_t kMaxWidth = 1ull << 30;              // 2 width lanes of the finalize stay below 2**32

static uint32_t column_groups(uint64_t rows, uint64_t width) {
    uint64_t groups = rows < kColumnGroups ? rows : kColumnGroups;
    const uint64_t most = kMaxPartials / (2u * sizeof(float) * width);
    if (groups > most) groups = most;
    return groups < 1 ? 1u : (uint32_t)groups;
}

template <class T>
static void launch_forward(const NormForward &a, int edge, hipStream_t s) {
    const dim3 grid(strided_grid(a.rows, kBlock)), block(kBlock);
    if (edge == kNone) norm_rows_kernel<T, kNone><<<grid, block, 0, s>>>(a);
    else if (edge == kAdd) norm_rows_kernel<T, kAdd><<<grid, block, 0, s>>>(a);
    else norm_rows_kernel<T, kDropAdd><<<grid, block, 0, s>>>(a);
}

template <class T>
static void launch_backward(const NormBackward &a, int edge, bool columns, hipStream_t s) {
    const dim3 grid(strided_grid(a.rows, kBlock)), block(kBlock);
    if (edge == kNone) norm_rows_backward_kernel<T, kNone><<<grid, block, 0, s>>>(a);
    else if (edge == kAdd) norm_rows_backward_kernel<T, kAdd><<<grid, block, 0, s>>>(a);
    else norm_rows_backward_kernel<T, kDropAdd><<<grid, block, 0, s>>>(a);
    if (columns) {
        const dim3 tiles((a.width + kBlock - 1) / kBlock, column_groups(a.rows, a.width));
        norm_columns_kernel<T><<<tiles, block, 0, s>>>(a);
    }
}

template <class T>
static void launch_finalize(const NormBackward &a, uint32_t groups, void *dw, void *db, hipStream_t s) {
    const dim3 grid((unsigned)((2u * (uint64_t)a.width + kBlock - 1) / kBlock));
    norm_finalize_kernel<T><<<grid, dim3(kBlock), 0, s>>>(a.partials, groups, a.width,
                                                          static_cast<typename T::raw *>(dw),
                                                          static_cast<typename T::raw *>(db));
}

template <class T>
static void launch_dropout(const void *x, void *y, uint64_t n, const Mask &mask, hipStream_t s) {
    const dim3 grid(strided_grid(((n + 7) / 8 + kBlock - 1) / kBlock, kBlock));
    dropout_kernel<T><<<grid, dim3(kBlock), 0, s>>>(static_cast<const typename T::raw *>(x),
                                                    static_cast<typename T::raw *>(y), n, mask);
}

// ---- argument checks --------------------------------------------------------------------------------
static bool half_or_float(int32_t dtype) { return dtype == NT_F32 || dtype == NT_F16 || dtype == NT_BF16; }

static int32_t check_rows(const char *entry, int32_t dtype, int32_t weight_dtype, bool has_params, uint64_t rows,
                          uint64_t width, uint32_t threshold) {
    const std::string name(entry);
    if (!half_or_float(dtype)) return fail(NT_ERR_TYPE, name + ": activations must be float32, float16 or bfloat16");
    if (has_params && weight_dtype != dtype && weight_dtype != NT_F32)
        return fail(NT_ERR_TYPE, name + ": weight and bias must have the activations' dtype or float32");
    if (width == 0 || width > kMaxWidth) return fail(NT_ERR_VALUE, name + ": the width must be 1..2**30");
    if (rows > 0xffffffffffffull / width) return fail(NT_ERR_VALUE, name + ": too many elements");
    if (threshold > 65536u) return fail(NT_ERR_VALUE, name + ": the drop threshold must be 0..65536");
    return NT_OK;
}

// One array argument: `count` elements of `dtype`, written or only read.
struct Array {
    const void *ptr;
    int32_t dtype;
    uint64_t count;
    bool written, needed;
};

// Needed arrays are there, all are aligned to their dtype, and what is
// written overlaps nothing else.
static int32_t check_arrays(const char *entry, std::initializer_list<Array> arrays) {
    for (const Array &a : arrays) {
        const uint64_t size = a.dtype == NT_F32 ? 4u : 2u;
        if (a.ptr == nullptr) {
            if (a.needed) return fail(NT_ERR_VALUE, std::string(entry) + ": NULL array");
            continue;
        }
        const uintptr_t start = (uintptr_t)a.ptr;
        if (start % size != 0) return fail(NT_ERR_VALUE, std::string(entry) + ": an array is not aligned to its dtype");
        if (!a.written) continue;
        for (const Array &b : arrays) {
            if (&a == &b || b.ptr == nullptr) continue;
            const uintptr_t other = (uintptr_t)b.ptr;
            if (start < other + b.count * (b.dtype == NT_F32 ? 4u : 2u) && other < start + a.count * size)
                return fail(NT_ERR_VALUE, std::string(entry) + ": an output overlaps another array");
        }
    }
    return NT_OK;
}

static int32_t forward(const char *entry, int32_t device, const NormForward &a, int32_t dtype, int edge, void *stream) {
    if ((a.mean == nullptr) != (a.rstd == nullptr))
        return fail(NT_ERR_VALUE, std::string(entry) + ": mean and rstd are given together");
    if (a.rows == 0) return NT_OK;
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case NT_F32: launch_forward<TF32>(a, edge, s); break;
        case NT_F16: launch_forward<TF16>(a, edge, s); break;
        default: launch_forward<TBF16>(a, edge, s); break;
    }
    NT_LAUNCH_CHECK("norm_rows_kernel launch");
    return NT_OK;
}

static int32_t backward(const char *entry, int32_t device, NormBackward a, int32_t dtype, int edge, void *dw, void *db,
                        void *stream) {
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    hipStream_t s = (hipStream_t)stream;
    const bool columns = dw != nullptr || db != nullptr;
    const uint32_t groups = column_groups(a.rows, a.width);
    void *workspace = nullptr;
    if (columns) {
        // The workspace goes back to the pool as soon as the kernels are queued: the pool reuses it on this
        // stream only.  Captured work would keep using it after that.
        int32_t capturing = 0;
        const int32_t queried = nt_stream_capturing(stream, &capturing);
        if (queried != NT_OK) return queried;
        if (capturing)
            return fail(NT_ERR_RUNTIME, std::string(entry) + ": not supported in stream capture");
        std::string error;
        const int32_t rc = device_pool().allocate(device, (uint64_t)groups * 2u * a.width * sizeof(float), stream,
                                                  &workspace, error);
        if (rc != NT_OK) return fail(rc, error);
        a.partials = static_cast<float *>(workspace);
    }
    switch (dtype) {
        case NT_F32: launch_backward<TF32>(a, edge, columns, s); break;
        case NT_F16: launch_backward<TF16>(a, edge, columns, s); break;
        default: launch_backward<TBF16>(a, edge, columns, s); break;
    }
    hipError_t status = hipGetLastError();
    if (columns && status == hipSuccess) {
        switch (a.weight_dtype) {
            case NT_F32: launch_finalize<TF32>(a, groups, dw, db, s); break;
            case NT_F16: launch_finalize<TF16>(a, groups, dw, db, s); break;
            default: launch_finalize<TBF16>(a, groups, dw, db, s); break;
        }
        status = hipGetLastError();
    }
    if (workspace != nullptr) {
        std::string error;
        (void)device_pool().release(workspace, error);
    }
    return hip_check(status, "layer norm backward launch");
}

}  // namespace nt

using namespace nt;

extern "C" {

int32_t nt_layer_norm(int32_t device, const void *x, int32_t dtype, const void *weight, const void *bias,
                      int32_t weight_dtype, float eps, void *y, float *mean, float *rstd, uint64_t rows,
                      uint64_t width, void *stream) {
    clear_error();
    int32_t rc = check_rows("nt_layer_norm", dtype, weight_dtype, weight != nullptr || bias != nullptr, rows, width, 0);
    if (rc != NT_OK) return rc;
    if (rows == 0) return NT_OK;
    const uint64_t n = rows * width;
    rc = check_arrays("nt_layer_norm", {{x, dtype, n, false, true}, {weight, weight_dtype, width, false, false},
                                        {bias, weight_dtype, width, false, false}, {y, dtype, n, true, true},
                                        {mean, NT_F32, rows, true, false}, {rstd, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    const NormForward a{x, nullptr, weight, bias, nullptr, y, mean, rstd, rows, (uint32_t)width, weight_dtype, eps, {}};
    return forward("nt_layer_norm", device, a, dtype, kNone, stream);
}

int32_t nt_layer_norm_backward(int32_t device, const void *dy, const void *x, int32_t dtype, const float *mean,
                               const float *rstd, const void *weight, int32_t weight_dtype, void *dx, void *dweight,
                               void *dbias, uint64_t rows, uint64_t width, void *stream) {
    clear_error();
    int32_t rc = check_rows("nt_layer_norm_backward", dtype, weight_dtype,
                            weight != nullptr || dweight != nullptr || dbias != nullptr, rows, width, 0);
    if (rc != NT_OK) return rc;
    const uint64_t n = rows * width;
    const bool any = rows > 0;
    rc = check_arrays("nt_layer_norm_backward",
                      {{dy, dtype, n, false, any}, {x, dtype, n, false, any}, {mean, NT_F32, rows, false, any},
                       {rstd, NT_F32, rows, false, any}, {weight, weight_dtype, width, false, false},
                       {dx, dtype, n, true, any}, {dweight, weight_dtype, width, true, false},
                       {dbias, weight_dtype, width, true, false}});
    if (rc != NT_OK) return rc;
    const NormBackward a{dy, nullptr, x, weight, mean, rstd, dx, nullptr, nullptr, rows, (uint32_t)width, weight_dtype, {}};
    return backward("nt_layer_norm_backward", device, a, dtype, kNone, dweight, dbias, stream);
}

int32_t nt_dropout(int32_t device, const void *x, int32_t dtype, void *y, uint64_t count, uint32_t threshold,
                   uint64_t seed, uint64_t offset, void *stream) {
    clear_error();
    if (!half_or_float(dtype)) return fail(NT_ERR_TYPE, "nt_dropout: activations must be float32, float16 or bfloat16");
    if (threshold > 65536u) return fail(NT_ERR_VALUE, "nt_dropout: the drop threshold must be 0..65536");
    if (count == 0) return NT_OK;
    if (count > 0xffffffffffffull) return fail(NT_ERR_VALUE, "nt_dropout: too many elements");
    // In place (y == x) each lane reads its elements before it writes them.
    int32_t rc = check_arrays("nt_dropout", {{x, dtype, x == y ? 0 : count, false, true}, {y, dtype, count, true, true}});
    if (rc != NT_OK) return rc;
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    const Mask mask = make_mask(threshold, seed, offset);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case NT_F32: launch_dropout<TF32>(x, y, count, mask, s); break;
        case NT_F16: launch_dropout<TF16>(x, y, count, mask, s); break;
        default: launch_dropout<TBF16>(x, y, count, mask, s); break;
    }
    NT_LAUNCH_CHECK("dropout_kernel launch");
    return NT_OK;
}

int32_t nt_dropout_add_layer_norm(int32_t device, const void *x, const void *residual, int32_t dtype,
                                  const void *weight, const void *bias, int32_t weight_dtype, float eps,
                                  uint32_t threshold, uint64_t seed, uint64_t offset, void *total, void *y, float *mean,
                                  float *rstd, uint64_t rows, uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_dropout_add_layer_norm";
    int32_t rc = check_rows(entry, dtype, weight_dtype, weight != nullptr || bias != nullptr, rows, width, threshold);
    if (rc != NT_OK) return rc;
    if (rows == 0) return NT_OK;
    const uint64_t n = rows * width;
    rc = check_arrays(entry, {{x, dtype, n, false, true}, {residual, dtype, n, false, true},
                              {weight, weight_dtype, width, false, false}, {bias, weight_dtype, width, false, false},
                              {total, dtype, n, true, true}, {y, dtype, n, true, true},
                              {mean, NT_F32, rows, true, false}, {rstd, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    const NormForward a{x, residual, weight, bias, total, y, mean, rstd, rows, (uint32_t)width, weight_dtype, eps,
                        make_mask(threshold, seed, offset)};
    return forward(entry, device, a, dtype, threshold == 0 ? kAdd : kDropAdd, stream);
}

int32_t nt_dropout_add_layer_norm_backward(int32_t device, const void *dy, const void *dtotal, const void *total,
                                           int32_t dtype, const float *mean, const float *rstd, const void *weight,
                                           int32_t weight_dtype, uint32_t threshold, uint64_t seed, uint64_t offset,
                                           void *dx, void *dresidual, void *dweight, void *dbias, uint64_t rows,
                                           uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_dropout_add_layer_norm_backward";
    int32_t rc = check_rows(entry, dtype, weight_dtype, weight != nullptr || dweight != nullptr || dbias != nullptr,
                            rows, width, threshold);
    if (rc != NT_OK) return rc;
    const uint64_t n = rows * width;
    const bool any = rows > 0;
    rc = check_arrays(entry, {{dy, dtype, n, false, any}, {dtotal, dtype, n, false, false},
                              {total, dtype, n, false, any}, {mean, NT_F32, rows, false, any},
                              {rstd, NT_F32, rows, false, any}, {weight, weight_dtype, width, false, false},
                              {dx, dtype, n, true, any}, {dresidual, dtype, n, true, any},
                              {dweight, weight_dtype, width, true, false}, {dbias, weight_dtype, width, true, false}});
    if (rc != NT_OK) return rc;
    const NormBackward a{dy, dtotal, total, weight, mean, rstd, dx, dresidual, nullptr, rows, (uint32_t)width,
                         weight_dtype, make_mask(threshold, seed, offset)};
    return backward(entry, device, a, dtype, threshold == 0 ? kAdd : kDropAdd, dweight, dbias, stream);
}

}  // extern "C"
