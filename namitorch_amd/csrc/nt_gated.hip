// nt_gated.hip — the edge after a block that is normalized before and after
// it: the norm of the block's output, its gate, the residual stream's scale
// and sum, and the norm for the next block; with the backward pass.
//
// N(x; w, b) = (x - mean) rstd w + b is layer norm, or with mean 0 and rstd of
// the root mean square.  With s the residual's scale and a the gate:
//   n = N(x; u, k),   t = s r + a n,   y = N(t; w, b)
// and, with h and i the normalized t and x, g = dy w,
//   dt = rstd (g - sum g / W - h sum(g h) / W) + what t gets from elsewhere
//   dr = s dt,   da = dt n,   q = a dt u
//   dx = rstd' (q - sum q / W - i sum(q i) / W)
//   dw = sum dy h, db = sum dy, du = sum a dt i, dk = sum a dt  over rows
// (no sums of g and q where the norm takes no mean).
//
// The gate has a row for all rows, one for each run of rows (a sequence), or
// one for each row.  In the first two cases the sums over rows that du, dk and
// da need are the same two, sum(dt i) and sum(dt) of each run:
//   da = u sum(dt i) + k sum(dt),   du = a sum(dt i),   dk = a sum(dt),
// the last two added over the runs.
//
// Sums and statistics are float32 (a lane's share of a row 64 bits in the
// kernels for rows of any width), over rows in a fixed order; each result is
// rounded once.  y is of t before its rounding; the backward pass reads t.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "nt_entry.hpp"
#include "nt_internal.hpp"
#include "nt_pool.hpp"
#include "nt_row_ops.hpp"
#include "nt_rows.hpp"

namespace nt {

struct Gate {
    const void *at;             // may be null
    int32_t dtype;
    uint32_t runs;              // its rows
    uint64_t run;               // rows of the stream that share one
    __device__ __forceinline__ uint64_t row(uint64_t r) const { return runs == 1u ? 0u : r / run; }
};

struct GatedForward {
    const void *x, *residual, *inner_weight, *inner_bias, *weight, *bias;
    Gate gate;
    void *total, *y;
    float *inner_mean, *inner_rstd, *mean, *rstd;      // each may be null
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    float scale, eps;
};

struct GatedBackward {
    const void *dy, *dtotal, *x, *t, *inner_weight, *inner_bias, *weight;
    Gate gate;
    const float *inner_mean, *inner_rstd, *mean, *rstd;
    void *dx, *dresidual, *dgate;
    float *row_sums;            // [rows][2]: of g and g h over each row (rows of any width)
    float *partials;            // [blocks][4][width]: sums of dt i, dt, dy h, dy
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    float scale;
    uint32_t run_blocks;        // workgroups, or groups of rows, of each run
};

// Sum of a value of 64 bits over the workgroup, as float32 on every lane.
__device__ __forceinline__ float block_total(double v, double *shared) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    double total = 0.0;
    for (uint32_t k = 0; k < blockDim.x / 64u; ++k) total += shared[k];
    return (float)total;
}

// ---- rows of any width: a workgroup a row ----------------------------------------------------------
template <class T>
__device__ __forceinline__ float total_of(const GatedForward &a, uint64_t base, uint64_t gate_row, uint32_t c, float mean,
                                          float rstd) {
    const float x = load1<T>(reinterpret_cast<const typename T::raw *>(a.x), base + c);
    const float n = __builtin_fmaf((x - mean) * rstd, load_param(a.inner_weight, a.weight_dtype, c, 1.0f),
                                   load_param(a.inner_bias, a.weight_dtype, c, 0.0f));
    const float gate = load_param(a.gate.at, a.gate.dtype, gate_row * a.width + c, 1.0f);
    const float r = load1<T>(reinterpret_cast<const typename T::raw *>(a.residual), base + c);
    return __builtin_fmaf(gate, n, a.scale * r);
}

template <class T, bool RMS>
__global__ __launch_bounds__(kBlock) void gated_rows_kernel(GatedForward a) {
    __shared__ double shared[kBlock / 64];
    const float width = (float)a.width;
    const auto *x = reinterpret_cast<const typename T::raw *>(a.x);
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width, gate_row = a.gate.row(row);
        float means[2] = {0.0f, 0.0f}, rstds[2];
        const auto value = [&](int which, uint32_t c) {
            return which == 0 ? load1<T>(x, base + c) : total_of<T>(a, base, gate_row, c, means[0], rstds[0]);
        };
        for (int which = 0; which < 2; ++which) {
            if constexpr (!RMS) {
                double sum = 0.0;
                for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) sum += value(which, c);
                means[which] = block_total(sum, shared) / width;
            }
            double squares = 0.0;
            for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
                const float d = value(which, c) - means[which];
                squares = __builtin_fma((double)d, (double)d, squares);
            }
            rstds[which] = 1.0f / __builtin_sqrtf(block_total(squares, shared) / width + a.eps);
        }
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float t = value(1, c);
            store1<T>(reinterpret_cast<typename T::raw *>(a.total), base + c, t);
            store1<T>(reinterpret_cast<typename T::raw *>(a.y), base + c,
                      __builtin_fmaf((t - means[1]) * rstds[1], load_param(a.weight, a.weight_dtype, c, 1.0f),
                                     load_param(a.bias, a.weight_dtype, c, 0.0f)));
        }
        if (threadIdx.x == 0 && a.rstd != nullptr) {
            a.inner_rstd[row] = rstds[0];
            a.rstd[row] = rstds[1];
            if constexpr (!RMS) {
                a.inner_mean[row] = means[0];
                a.mean[row] = means[1];
            }
        }
    }
}

// dt of an element, from its row's sums of g and g h over W.
template <class T>
__device__ __forceinline__ float total_grad(const GatedBackward &a, uint64_t base, uint32_t c, float mean, float rstd,
                                            float level, float along) {
    const float g = load1<T>(reinterpret_cast<const typename T::raw *>(a.dy), base + c) *
                    load_param(a.weight, a.weight_dtype, c, 1.0f);
    const float h = (load1<T>(reinterpret_cast<const typename T::raw *>(a.t), base + c) - mean) * rstd;
    const float dt = rstd * (g - level - h * along);
    return a.dtotal == nullptr ? dt : dt + load1<T>(reinterpret_cast<const typename T::raw *>(a.dtotal), base + c);
}

template <class T, bool RMS>
__global__ __launch_bounds__(kBlock) void gated_rows_backward_kernel(GatedBackward a) {
    __shared__ double shared[kBlock / 64];
    const float width = (float)a.width;
    const auto *dy = reinterpret_cast<const typename T::raw *>(a.dy);
    const auto *t = reinterpret_cast<const typename T::raw *>(a.t);
    const auto *x = reinterpret_cast<const typename T::raw *>(a.x);
    const bool each = a.dgate != nullptr && a.gate.runs == a.rows;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width, gate_row = a.gate.row(row) * a.width;
        const float mean = RMS ? 0.0f : a.mean[row], rstd = a.rstd[row];
        const float inner_mean = RMS ? 0.0f : a.inner_mean[row], inner_rstd = a.inner_rstd[row];
        double levels = 0.0, alongs = 0.0;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float g = load1<T>(dy, base + c) * load_param(a.weight, a.weight_dtype, c, 1.0f);
            levels += g;
            alongs = __builtin_fma((double)g, (double)((load1<T>(t, base + c) - mean) * rstd), alongs);
        }
        const float along = block_total(alongs, shared) / width;
        const float level = RMS ? 0.0f : block_total(levels, shared) / width;
        if (threadIdx.x == 0) {
            a.row_sums[2 * row] = level;
            a.row_sums[2 * row + 1] = along;
        }
        levels = alongs = 0.0;
        const auto inner_grad = [&](uint32_t c, float dt) {
            return dt * load_param(a.gate.at, a.gate.dtype, gate_row + c, 1.0f) *
                   load_param(a.inner_weight, a.weight_dtype, c, 1.0f);
        };
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float q = inner_grad(c, total_grad<T>(a, base, c, mean, rstd, level, along));
            levels += q;
            alongs = __builtin_fma((double)q, (double)((load1<T>(x, base + c) - inner_mean) * inner_rstd), alongs);
        }
        const float inner_along = block_total(alongs, shared) / width;
        const float inner_level = RMS ? 0.0f : block_total(levels, shared) / width;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float dt = total_grad<T>(a, base, c, mean, rstd, level, along);
            const float i = (load1<T>(x, base + c) - inner_mean) * inner_rstd;
            store1<T>(reinterpret_cast<typename T::raw *>(a.dresidual), base + c, a.scale * dt);
            store1<T>(reinterpret_cast<typename T::raw *>(a.dx), base + c,
                      inner_rstd * (inner_grad(c, dt) - inner_level - i * inner_along));
            if (each) {
                const float n = __builtin_fmaf(i, load_param(a.inner_weight, a.weight_dtype, c, 1.0f),
                                               load_param(a.inner_bias, a.weight_dtype, c, 0.0f));
                store_param(a.dgate, a.gate.dtype, base + c, dt * n);
            }
        }
    }
}

// The four column sums over a group of a run's rows, one column a lane.
// Where each row has a gate of its own, dt is taken with it.
template <class T, bool RMS>
__global__ __launch_bounds__(kBlock) void gated_columns_kernel(GatedBackward a, uint32_t groups) {
    const uint32_t c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.width) return;
    const auto *dy = reinterpret_cast<const typename T::raw *>(a.dy);
    const auto *t = reinterpret_cast<const typename T::raw *>(a.t);
    const auto *x = reinterpret_cast<const typename T::raw *>(a.x);
    const bool each = a.gate.at != nullptr && a.gate.runs == a.rows && a.rows > 1;
    const uint64_t run = each ? a.rows : a.gate.run;
    for (uint32_t group = blockIdx.y; group < groups; group += gridDim.y) {
        const uint64_t first = group / a.run_blocks * run;
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint64_t r = group % a.run_blocks; r < run; r += a.run_blocks) {
            const uint64_t row = first + r, base = row * a.width;
            const float mean = RMS ? 0.0f : a.mean[row], rstd = a.rstd[row];
            float dt = total_grad<T>(a, base, c, mean, rstd, a.row_sums[2 * row], a.row_sums[2 * row + 1]);
            if (each) dt *= load_param(a.gate.at, a.gate.dtype, base + c, 1.0f);
            const float i = (load1<T>(x, base + c) - (RMS ? 0.0f : a.inner_mean[row])) * a.inner_rstd[row];
            const float g = load1<T>(dy, base + c);
            sums[0] = __builtin_fmaf(dt, i, sums[0]);
            sums[1] += dt;
            sums[2] = __builtin_fmaf(g, (load1<T>(t, base + c) - mean) * rstd, sums[2]);
            sums[3] += g;
        }
        float *out = a.partials + group * 4ull * a.width + c;
        for (int k = 0; k < 4; ++k) out[k * (uint64_t)a.width] = sums[k];
    }
}

// The vectors' gradients from the partial sums: 32 columns and 32 slices a
// workgroup.  A slice takes whole runs where there are several, else a share
// of the one run's blocks; slices are joined in order.
struct GatedVectors {
    void *inner_weight, *inner_bias, *gate, *weight, *bias;     // each may be null
};
constexpr uint32_t kVectorColumns = 32, kVectorSlices = 32;

__global__ __launch_bounds__(kVectorColumns * kVectorSlices) void gated_vectors_kernel(GatedBackward a, GatedVectors to,
                                                                                        uint32_t runs, bool each) {
    __shared__ float shared[4][kVectorSlices][kVectorColumns + 1];
    const uint32_t column = threadIdx.x % kVectorColumns, slice = threadIdx.x / kVectorColumns;
    const uint32_t c = blockIdx.x * kVectorColumns + column;
    const uint64_t line = a.width, block = 4u * line;
    const bool there = c < a.width;
    const float u = there ? load_param(a.inner_weight, a.weight_dtype, c, 1.0f) : 0.0f;
    const float k = there ? load_param(a.inner_bias, a.weight_dtype, c, 0.0f) : 0.0f;
    const auto gate_of = [&](uint32_t run) {
        return each ? 1.0f : load_param(a.gate.at, a.gate.dtype, run * line + c, 1.0f);
    };
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (there && runs == 1u) {
        for (uint32_t b = slice; b < a.run_blocks; b += kVectorSlices)
            for (int v = 0; v < 4; ++v) sums[v] += a.partials[b * block + v * line + c];
    } else if (there) {
        for (uint32_t run = slice; run < runs; run += kVectorSlices) {
            float own[2] = {0.0f, 0.0f};
            for (uint32_t b = run * a.run_blocks; b < (run + 1u) * a.run_blocks; ++b) {
                own[0] += a.partials[b * block + c];
                own[1] += a.partials[b * block + line + c];
                sums[2] += a.partials[b * block + 2u * line + c];
                sums[3] += a.partials[b * block + 3u * line + c];
            }
            if (to.gate != nullptr)
                store_param(to.gate, a.gate.dtype, run * line + c, __builtin_fmaf(u, own[0], k * own[1]));
            const float gate = gate_of(run);
            sums[0] = __builtin_fmaf(gate, own[0], sums[0]);
            sums[1] = __builtin_fmaf(gate, own[1], sums[1]);
        }
    }
    for (int v = 0; v < 4; ++v) shared[v][slice][column] = sums[v];
    __syncthreads();
    if (slice >= 4u || !there) return;
    float sum = 0.0f;
    for (uint32_t s = 0; s < kVectorSlices; ++s) sum += shared[slice][s][column];
    const float gate = runs == 1u ? gate_of(0) : 1.0f;
    void *out = slice == 0u ? to.inner_weight : slice == 1u ? to.inner_bias : slice == 2u ? to.weight : to.bias;
    if (out != nullptr) store_param(out, a.weight_dtype, c, slice < 2u ? sum * gate : sum);
    if (runs != 1u || each || to.gate == nullptr || slice != 0u) return;
    float other = 0.0f;
    for (uint32_t s = 0; s < kVectorSlices; ++s) other += shared[1][s][column];
    store_param(to.gate, a.gate.dtype, c, __builtin_fmaf(u, sum, k * other));
}

// ---- launches ----------------------------------------------------------------------------------------
constexpr uint32_t kMostBlocks = 8192;
constexpr uint32_t kRunGroups = 256;                    // groups of rows of the column sums, over all runs
constexpr uint64_t kMostWidth = 1ull << 24;

template <class T>
static void launch_gated(const GatedForward &a, bool rms, hipStream_t s) {
    const dim3 grid((unsigned)std::min<uint64_t>(a.rows, kMostBlocks));
    if (rms) gated_rows_kernel<T, true><<<grid, dim3(kBlock), 0, s>>>(a);
    else gated_rows_kernel<T, false><<<grid, dim3(kBlock), 0, s>>>(a);
}

template <class T>
static void launch_gated_backward(const GatedBackward &a, bool rms, uint32_t groups, hipStream_t s) {
    const dim3 grid((unsigned)std::min<uint64_t>(a.rows, kMostBlocks));
    const dim3 columns((a.width + kBlock - 1) / kBlock, std::min(groups, 65535u));
    if (rms) gated_rows_backward_kernel<T, true><<<grid, dim3(kBlock), 0, s>>>(a);
    else gated_rows_backward_kernel<T, false><<<grid, dim3(kBlock), 0, s>>>(a);
    if (rms) gated_columns_kernel<T, true><<<columns, dim3(kBlock), 0, s>>>(a, groups);
    else gated_columns_kernel<T, false><<<columns, dim3(kBlock), 0, s>>>(a, groups);
}

static int32_t check_gated(const char *entry, int32_t dtype, int32_t weight_dtype, bool has_params, const void *gate,
                           int32_t gate_dtype, uint64_t gate_rows, uint64_t rows, uint64_t width) {
    const std::string name(entry);
    if (!half_or_float(dtype)) return fail(NT_ERR_TYPE, name + ": activations must be float32, float16 or bfloat16");
    if (has_params && weight_dtype != dtype && weight_dtype != NT_F32)
        return fail(NT_ERR_TYPE, name + ": weights and biases must have the activations' dtype or float32");
    if (gate != nullptr && gate_dtype != dtype && gate_dtype != NT_F32)
        return fail(NT_ERR_TYPE, name + ": the gate must have the activations' dtype or float32");
    if (width == 0 || width > kMostWidth) return fail(NT_ERR_VALUE, name + ": the width must be 1..2**24");
    if (rows > 0xffffffffffffull / width || rows >= 1ull << 31)
        return fail(NT_ERR_VALUE, name + ": too many rows or elements");
    if (gate != nullptr && rows > 0 && (gate_rows == 0 || rows % gate_rows != 0))
        return fail(NT_ERR_VALUE, name + ": the gate's rows must divide the rows");
    return NT_OK;
}

}  // namespace nt

using namespace nt;

extern "C" {

int32_t nt_norm_gate_add_norm(int32_t device, const void *x, const void *residual, int32_t dtype,
                              const void *inner_weight, const void *inner_bias, const void *gate, int32_t gate_dtype,
                              uint64_t gate_rows, const void *weight, const void *bias, int32_t weight_dtype,
                              float residual_scale, float eps, int32_t rms, void *total, void *y, float *inner_mean,
                              float *inner_rstd, float *mean, float *rstd, uint64_t rows, uint64_t width,
                              void *stream) {
    clear_error();
    const char *entry = "nt_norm_gate_add_norm";
    const bool params = inner_weight != nullptr || inner_bias != nullptr || weight != nullptr || bias != nullptr;
    int32_t rc = check_gated(entry, dtype, weight_dtype, params, gate, gate_dtype, gate_rows, rows, width);
    if (rc != NT_OK) return rc;
    if (rows == 0) return NT_OK;
    const uint64_t n = rows * width;
    rc = check_arrays(entry, {{x, dtype, n, false, true}, {residual, dtype, n, false, true},
                              {inner_weight, weight_dtype, width, false, false},
                              {inner_bias, weight_dtype, width, false, false},
                              {gate, gate_dtype, gate_rows * width, false, false},
                              {weight, weight_dtype, width, false, false}, {bias, weight_dtype, width, false, false},
                              {total, dtype, n, true, true}, {y, dtype, n, true, true},
                              {inner_mean, NT_F32, rows, true, false}, {inner_rstd, NT_F32, rows, true, false},
                              {mean, NT_F32, rows, true, false}, {rstd, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    const bool stats = rstd != nullptr;
    if ((inner_rstd != nullptr) != stats || (inner_mean != nullptr) != (stats && !rms) ||
        (mean != nullptr) != (stats && !rms))
        return fail(NT_ERR_VALUE, std::string(entry) + ": statistics are given together, means where the norm has them");
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    const uint64_t runs = gate == nullptr ? 1u : gate_rows;
    const GatedForward a{x, residual, inner_weight, inner_bias, weight, bias,
                         {gate, gate_dtype, (uint32_t)runs, rows / runs}, total, y, inner_mean, inner_rstd, mean, rstd,
                         rows, (uint32_t)width, weight_dtype, residual_scale, eps};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case NT_F32: launch_gated<TF32>(a, rms != 0, s); break;
        case NT_F16: launch_gated<TF16>(a, rms != 0, s); break;
        default: launch_gated<TBF16>(a, rms != 0, s); break;
    }
    NT_LAUNCH_CHECK("gated norm launch");
    return NT_OK;
}

int32_t nt_norm_gate_add_norm_backward(int32_t device, const void *dy, const void *dtotal, const void *x,
                                       const void *total, int32_t dtype, const float *inner_mean,
                                       const float *inner_rstd, const float *mean, const float *rstd,
                                       const void *inner_weight, const void *inner_bias, const void *gate,
                                       int32_t gate_dtype, uint64_t gate_rows, const void *weight, int32_t weight_dtype,
                                       float residual_scale, void *dx, void *dresidual, void *dinner_weight,
                                       void *dinner_bias, void *dgate, void *dweight, void *dbias, uint64_t rows,
                                       uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_norm_gate_add_norm_backward";
    const bool params = inner_weight != nullptr || inner_bias != nullptr || weight != nullptr ||
                        dinner_weight != nullptr || dinner_bias != nullptr || dweight != nullptr || dbias != nullptr;
    int32_t rc = check_gated(entry, dtype, weight_dtype, params, gate, gate_dtype, gate_rows, rows, width);
    if (rc != NT_OK) return rc;
    if (gate == nullptr && dgate != nullptr) return fail(NT_ERR_VALUE, std::string(entry) + ": there is no gate");
    const uint64_t n = rows * width, gate_size = gate == nullptr ? 0 : gate_rows * width;
    const bool any = rows > 0;
    rc = check_arrays(entry, {{dy, dtype, n, false, any}, {dtotal, dtype, n, false, false}, {x, dtype, n, false, any},
                              {total, dtype, n, false, any}, {inner_mean, NT_F32, rows, false, false},
                              {inner_rstd, NT_F32, rows, false, any}, {mean, NT_F32, rows, false, false},
                              {rstd, NT_F32, rows, false, any}, {inner_weight, weight_dtype, width, false, false},
                              {inner_bias, weight_dtype, width, false, false}, {gate, gate_dtype, gate_size, false, false},
                              {weight, weight_dtype, width, false, false}, {dx, dtype, n, true, any},
                              {dresidual, dtype, n, true, any}, {dinner_weight, weight_dtype, width, true, false},
                              {dinner_bias, weight_dtype, width, true, false}, {dgate, gate_dtype, gate_size, true, false},
                              {dweight, weight_dtype, width, true, false}, {dbias, weight_dtype, width, true, false}});
    if (rc != NT_OK) return rc;
    if ((inner_mean != nullptr) != (mean != nullptr))
        return fail(NT_ERR_VALUE, std::string(entry) + ": both means are given or none");
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    rc = refuse_capture(entry, stream);
    if (rc != NT_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (!any) {
        for (void *vector : {dinner_weight, dinner_bias, dweight, dbias})
            if (vector != nullptr && (rc = nt_fill(vector, width, weight_dtype == NT_F32 ? 4 : 2, 0, stream)) != NT_OK)
                return rc;
        return dgate == nullptr ? NT_OK : nt_fill(dgate, gate_size, gate_dtype == NT_F32 ? 4 : 2, 0, stream);
    }
    const bool rms = mean == nullptr, each = gate != nullptr && gate_rows == rows && rows > 1;
    const uint64_t gate_runs = gate == nullptr ? 1u : gate_rows;
    const uint32_t runs = each ? 1u : (uint32_t)gate_runs;          // whose sums are kept apart
    GatedBackward a{dy, dtotal, x, total, inner_weight, inner_bias, weight,
                    {gate, gate_dtype, (uint32_t)gate_runs, rows / gate_runs}, inner_mean, inner_rstd, mean, rstd,
                    dx, dresidual, each ? dgate : nullptr, nullptr, nullptr, rows, (uint32_t)width, weight_dtype,
                    residual_scale, 1};
    a.run_blocks = (uint32_t)std::min<uint64_t>(rows / runs, std::max(1u, kRunGroups / runs));
    Workspace room;
    room.want(&a.row_sums, 2u * rows);
    room.want(&a.partials, 4ull * width * runs * a.run_blocks);
    rc = room.allocate(device, stream);
    if (rc != NT_OK) return rc;
    const uint32_t groups = runs * a.run_blocks;
    switch (dtype) {
        case NT_F32: launch_gated_backward<TF32>(a, rms, groups, s); break;
        case NT_F16: launch_gated_backward<TF16>(a, rms, groups, s); break;
        default: launch_gated_backward<TBF16>(a, rms, groups, s); break;
    }
    const GatedVectors vectors{dinner_weight, dinner_bias, each ? nullptr : dgate, dweight, dbias};
    gated_vectors_kernel<<<dim3((unsigned)((width + kVectorColumns - 1) / kVectorColumns)),
                           dim3(kVectorColumns * kVectorSlices), 0, s>>>(a, vectors, runs, each);
    return hip_check(hipGetLastError(), "gated norm backward launch");
}

}  // extern "C"
