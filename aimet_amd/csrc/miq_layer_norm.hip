// Layer norm for gfx950: forward, and the backward pass with the reductions of the weight's and the bias' gradient.
//
//   m = mean(x), v = mean((x - m)^2), r = 1 / sqrt(v + eps), xhat = (x - m) r, y = xhat w + b
//   gw = g w, dx = r (gw - mean(gw) - xhat mean(gw xhat)), dw = sum over rows of g xhat, db = sum over rows of g
//
// All arithmetic is float32; only what is stored in bfloat16 is rounded to it, once.
#include "miq_io.h"

#include <algorithm>
#include <type_traits>

namespace miq
{
namespace
{
// sum over the block, the same in every thread; `lds` holds kBlock / 64 floats and may be used again after the next barrier
__device__ __forceinline__ float block_sum(float v, float* lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kBlock / 64; ++i)
        s += lds[i];
    return s;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void ln_fwd_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                        const T* __restrict__ b, int64_t width, float eps,
                                                        T* __restrict__ y, float* __restrict__ mean,
                                                        float* __restrict__ rstd)
{
    using IO = IOTraits<T>;
    __shared__ float lds[kBlock / 64];
    const int64_t row = blockIdx.x;
    const T* px       = x + row * width;
    float s           = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kBlock)
        s += IO::load1(px + c);
    const float m = block_sum(s, lds) / (float) width;
    float q       = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kBlock)
    {
        const float d = IO::load1(px + c) - m;
        q += d * d;
    }
    const float r = 1.0f / sqrtf(block_sum(q, lds) / (float) width + eps);
    for (int64_t c = threadIdx.x; c < width; c += kBlock)
    {
        const float h = (IO::load1(px + c) - m) * r;
        IO::store1(y + row * width + c, h * (w ? IO::load1(w + c) : 1.f) + (b ? IO::load1(b + c) : 0.f));
    }
    if (threadIdx.x == 0 && mean)
    {
        mean[row] = m;
        rstd[row] = r;
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void ln_dx_kernel(const T* __restrict__ x, const T* __restrict__ g,
                                                       const T* __restrict__ w, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, int64_t width,
                                                       T* __restrict__ dx)
{
    using IO = IOTraits<T>;
    __shared__ float lds[kBlock / 64];
    const int64_t row = blockIdx.x;
    const T* px       = x + row * width;
    const T* pg       = g + row * width;
    const float m = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kBlock)
    {
        const float gw = IO::load1(pg + c) * (w ? IO::load1(w + c) : 1.f);
        s1 += gw;
        s2 += gw * ((IO::load1(px + c) - m) * r);
    }
    const float m1 = block_sum(s1, lds) / (float) width;
    const float m2 = block_sum(s2, lds) / (float) width;
    for (int64_t c = threadIdx.x; c < width; c += kBlock)
    {
        const float gw = IO::load1(pg + c) * (w ? IO::load1(w + c) : 1.f);
        const float h  = (IO::load1(px + c) - m) * r;
        IO::store1(dx + row * width + c, r * (gw - m1 - h * m2));
    }
}

// column sums of a slice of the rows: partial[slice][0][c] = sum g xhat, partial[slice][1][c] = sum g
template <typename T>
__global__ __launch_bounds__(kBlock) void ln_dparams_kernel(const T* __restrict__ x, const T* __restrict__ g,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, int64_t rows,
                                                            int64_t width, int64_t rows_per_slice,
                                                            float* __restrict__ partial)
{
    using IO        = IOTraits<T>;
    const int64_t c = (int64_t) blockIdx.x * kBlock + threadIdx.x;
    if (c >= width)
        return;
    const int64_t first = blockIdx.y * rows_per_slice;
    const int64_t last  = first + rows_per_slice < rows ? first + rows_per_slice : rows;
    float sw = 0.f, sb = 0.f;
    for (int64_t row = first; row < last; ++row)
    {
        const float gv = IO::load1(g + row * width + c);
        sw += gv * ((IO::load1(x + row * width + c) - mean[row]) * rstd[row]);
        sb += gv;
    }
    partial[((int64_t) blockIdx.y * 2) * width + c]     = sw;
    partial[((int64_t) blockIdx.y * 2 + 1) * width + c] = sb;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void ln_join_kernel(const float* __restrict__ partial, int64_t slices,
                                                         int64_t width, T* __restrict__ dw, T* __restrict__ db)
{
    const int64_t c = (int64_t) blockIdx.x * kBlock + threadIdx.x;
    if (c >= width)
        return;
    T* out = blockIdx.y == 0 ? dw : db;
    if (!out)
        return;
    float s = 0.f;
    for (int64_t k = 0; k < slices; ++k)
        s += partial[(k * 2 + blockIdx.y) * width + c];
    IOTraits<T>::store1(out + c, s);
}

int64_t ln_slices(int64_t rows, int64_t width)
{
    const int64_t columns = (width + kBlock - 1) / kBlock;
    return std::max<int64_t>(1, std::min<int64_t>((1024 + columns - 1) / columns, rows / 16));
}

int check_shape(int64_t rows, int64_t width)
{
    MIQ_CHECK_ARG(rows >= 0 && width >= 1, "rows must not be negative and width must be positive");
    MIQ_CHECK_ARG(rows <= INT32_MAX && width <= INT32_MAX, "rows and width must be below 2^31");
    return MIQ_OK;
}

template <typename T>
int layer_norm_fwd(const T* x, const T* w, const T* b, int64_t rows, int64_t width, float eps, T* y, float* mean,
                   float* rstd, void* stream)
{
    if (int rc = check_shape(rows, width))
        return rc;
    if (rows == 0)
        return MIQ_OK;
    MIQ_CHECK_ARG(x && y, "null pointer");
    MIQ_CHECK_ARG((mean != nullptr) == (rstd != nullptr), "mean and rstd go together");
    hipLaunchKernelGGL(ln_fwd_kernel<T>, dim3((unsigned) rows), dim3(kBlock), 0, (hipStream_t) stream, x, w, b, width,
                       eps, y, mean, rstd);
    MIQ_CHECK_LAUNCH();
    return MIQ_OK;
}

template <typename T>
int layer_norm_bwd(const T* x, const T* g, const T* w, const float* mean, const float* rstd, int64_t rows,
                   int64_t width, T* dx, T* dw, T* db, float* workspace, void* stream)
{
    if (int rc = check_shape(rows, width))
        return rc;
    MIQ_CHECK_ARG(rows == 0 || (x && g && mean && rstd), "null pointer");
    MIQ_CHECK_ARG(!(dw || db) || workspace, "the gradients of weight and bias need the workspace");
    hipStream_t s = (hipStream_t) stream;
    if (dx && rows)
    {
        hipLaunchKernelGGL(ln_dx_kernel<T>, dim3((unsigned) rows), dim3(kBlock), 0, s, x, g, w, mean, rstd, width, dx);
        MIQ_CHECK_LAUNCH();
    }
    if (dw || db)
    {
        const int64_t slices = ln_slices(rows, width), columns = (width + kBlock - 1) / kBlock;
        hipLaunchKernelGGL(ln_dparams_kernel<T>, dim3((unsigned) columns, (unsigned) slices), dim3(kBlock), 0, s, x, g,
                           mean, rstd, rows, width, (rows + slices - 1) / slices, workspace);
        MIQ_CHECK_LAUNCH();
        hipLaunchKernelGGL(ln_join_kernel<T>, dim3((unsigned) columns, 2), dim3(kBlock), 0, s, workspace, slices,
                           width, dw, db);
        MIQ_CHECK_LAUNCH();
    }
    return MIQ_OK;
}
}   // namespace
}   // namespace miq

using namespace miq;

extern "C"
{
int64_t miq_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width)
{
    if (rows < 0 || width < 1)
        return 0;
    return ln_slices(rows, width) * 2 * width * (int64_t) sizeof(float);
}

int miq_layer_norm_fwd_f32(const float* x, const float* weight, const float* bias, int64_t rows, int64_t width,
                           float eps, float* y, float* mean, float* rstd, void* stream)
{
    return layer_norm_fwd(x, weight, bias, rows, width, eps, y, mean, rstd, stream);
}

int miq_layer_norm_fwd_bf16(const uint16_t* x, const uint16_t* weight, const uint16_t* bias, int64_t rows,
                            int64_t width, float eps, uint16_t* y, float* mean, float* rstd, void* stream)
{
    return layer_norm_fwd(x, weight, bias, rows, width, eps, y, mean, rstd, stream);
}

int miq_layer_norm_bwd_f32(const float* x, const float* grad, const float* weight, const float* mean,
                           const float* rstd, int64_t rows, int64_t width, float* dx, float* dweight, float* dbias,
                           void* workspace, void* stream)
{
    return layer_norm_bwd(x, grad, weight, mean, rstd, rows, width, dx, dweight, dbias, (float*) workspace, stream);
}

int miq_layer_norm_bwd_bf16(const uint16_t* x, const uint16_t* grad, const uint16_t* weight, const float* mean,
                            const float* rstd, int64_t rows, int64_t width, uint16_t* dx, uint16_t* dweight,
                            uint16_t* dbias, void* workspace, void* stream)
{
    return layer_norm_bwd(x, grad, weight, mean, rstd, rows, width, dx, dweight, dbias, (float*) workspace, stream);
}
}   // extern "C"
