// Matrix product with bias, activation and residual in its epilogue, and its backward pass, for gfx950.
//
//   z = x w^T + b, y = act(z) + residual                          x [rows, in], w [out, in], y [rows, out]
//   dz = g act'(z), dx = dz w, dw = dz^T x, db = sum over rows of dz, dresidual = g
#include "miq_activation.h"
#include "miq_io.h"

#include <algorithm>
#include <type_traits>

namespace miq
{
namespace
{
// What the backward pass keeps of z = x w^T + b.  float32 tensors keep it as it is.  bfloat16 ones keep a half: as
// many bytes, three bits more, and z matters only through act'(z), which is flat far out, so saturating at the
// largest half loses nothing.  A z > 0 too small for a half is kept as the smallest one: ReLU's derivative goes by
// its sign.  NaN stays NaN.
template <typename T>
using Saved = std::conditional_t<std::is_same<T, float>::value, float, _Float16>;

__device__ __forceinline__ void save_z(float* p, float z)
{
    *p = z;
}
__device__ __forceinline__ void save_z(_Float16* p, float z)
{
    const float c = z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z;
    *p            = (_Float16) (z > 0.f && z < 0x1p-24f ? 0x1p-24f : c);
}

constexpr int kTile = 64, kDeep = 16;

// C[m, n] = sum over k of A(m, k) B(n, k): A(m, k) = a[m * ams + k * aks], B likewise.
// One 64 x 64 tile of C in a block of 256 threads, 4 x 4 values in each, operands through LDS in float32.
template <typename T, int ACT>
__global__ __launch_bounds__(kBlock) void product_kernel(const T* __restrict__ a, int64_t ams, int64_t aks,
                                                         const T* __restrict__ b, int64_t bns, int64_t bks, int64_t m,
                                                         int64_t n, int64_t k, const T* __restrict__ bias,
                                                         const T* __restrict__ residual, T* __restrict__ c,
                                                         Saved<T>* __restrict__ saved)
{
    using IO = IOTraits<T>;
    __shared__ float la[kDeep][kTile + 4], lb[kDeep][kTile + 4];
    const int64_t tiles_n = (n + kTile - 1) / kTile;
    const int64_t m0 = (blockIdx.x / tiles_n) * kTile, n0 = (blockIdx.x % tiles_n) * kTile;
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += kDeep)
    {
        for (int i = threadIdx.x; i < kTile * kDeep; i += kBlock)
        {
            const int kk = i % kDeep, r = i / kDeep;
            la[kk][r] = m0 + r < m && k0 + kk < k ? IO::load1(a + (m0 + r) * ams + (k0 + kk) * aks) : 0.f;
            lb[kk][r] = n0 + r < n && k0 + kk < k ? IO::load1(b + (n0 + r) * bns + (k0 + kk) * bks) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kDeep; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(la[kk][tm * 4 + i], lb[kk][tn * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
        {
            const int64_t r = m0 + tm * 4 + i, q = n0 + tn * 4 + j;
            if (r >= m || q >= n)
                continue;
            const float z = acc[i][j] + (bias ? IO::load1(bias + q) : 0.f);
            if (saved)
                save_z(saved + r * n + q, z);
            IO::store1(c + r * n + q, act_value<ACT>(z) + (residual ? IO::load1(residual + r * n + q) : 0.f));
        }
}

// dz = g act'(z) and its column sums over a slice of the rows
template <typename T, int ACT>
__global__ __launch_bounds__(kBlock) void slope_kernel(const T* __restrict__ g, const Saved<T>* __restrict__ z,
                                                       int64_t rows, int64_t cols, int64_t rows_per_slice,
                                                       T* __restrict__ dz, float* __restrict__ partial)
{
    using IO        = IOTraits<T>;
    const int64_t c = (int64_t) blockIdx.x * kBlock + threadIdx.x;
    if (c >= cols)
        return;
    const int64_t first = blockIdx.y * rows_per_slice;
    const int64_t last  = first + rows_per_slice < rows ? first + rows_per_slice : rows;
    float sum           = 0.f;
    for (int64_t r = first; r < last; ++r)
    {
        float d = IO::load1(g + r * cols + c);
        if (ACT != MIQ_ACT_NONE)
        {
            d *= act_slope<ACT>((float) z[r * cols + c]);
            IO::store1(dz + r * cols + c, d);
        }
        sum += d;
    }
    partial[(int64_t) blockIdx.y * cols + c] = sum;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void join_columns_kernel(const float* __restrict__ partial, int64_t slices,
                                                              int64_t cols, T* __restrict__ out)
{
    const int64_t c = (int64_t) blockIdx.x * kBlock + threadIdx.x;
    if (c >= cols)
        return;
    float s = 0.f;
    for (int64_t k = 0; k < slices; ++k)
        s += partial[k * cols + c];
    IOTraits<T>::store1(out + c, s);
}

template <typename F>
void with_activation(int activation, F&& f)
{
    switch (activation)
    {
    case MIQ_ACT_RELU: f(std::integral_constant<int, MIQ_ACT_RELU>()); break;
    case MIQ_ACT_SILU: f(std::integral_constant<int, MIQ_ACT_SILU>()); break;
    case MIQ_ACT_GELU: f(std::integral_constant<int, MIQ_ACT_GELU>()); break;
    case MIQ_ACT_GELU_TANH: f(std::integral_constant<int, MIQ_ACT_GELU_TANH>()); break;
    default: f(std::integral_constant<int, MIQ_ACT_NONE>()); break;
    }
}

int64_t slope_slices(int64_t rows, int64_t cols)
{
    const int64_t columns = (cols + kBlock - 1) / kBlock;
    return std::max<int64_t>(1, std::min<int64_t>((1024 + columns - 1) / columns, rows / 16));
}

int64_t up256(int64_t n)
{
    return (n + 255) / 256 * 256;
}

int check_shape(int64_t rows, int64_t in, int64_t out, int activation)
{
    MIQ_CHECK_ARG(rows >= 0 && in >= 0 && out >= 0, "rows, in_features and out_features must not be negative");
    MIQ_CHECK_ARG(rows <= INT32_MAX && in <= INT32_MAX && out <= INT32_MAX, "a size is 2^31 or more");
    MIQ_CHECK_ARG(activation >= MIQ_ACT_NONE && activation <= MIQ_ACT_GELU_TANH, "unknown activation %d", activation);
    return MIQ_OK;
}

template <typename T, int ACT>
int product(const T* a, int64_t ams, int64_t aks, const T* b, int64_t bns, int64_t bks, int64_t m, int64_t n,
            int64_t k, const T* bias, const T* residual, T* c, Saved<T>* saved, hipStream_t s)
{
    const int64_t tiles = ((m + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
    if (tiles == 0)
        return MIQ_OK;
    MIQ_CHECK_ARG(tiles <= INT32_MAX, "the product has too many tiles");
    hipLaunchKernelGGL((product_kernel<T, ACT>), dim3((unsigned) tiles), dim3(kBlock), 0, s, a, ams, aks, b, bns, bks,
                       m, n, k, bias, residual, c, saved);
    MIQ_CHECK_LAUNCH();
    return MIQ_OK;
}

template <typename T>
int64_t workspace_bytes(int64_t rows, int64_t in, int64_t out, int activation, int backward)
{
    (void) in;
    if (!backward)
        return 0;
    return (activation == MIQ_ACT_NONE ? 0 : up256(rows * out * (int64_t) sizeof(T))) +
           up256(slope_slices(rows, out) * out * (int64_t) sizeof(float));
}

template <typename T>
int linear_fwd(const T* x, const T* w, const T* bias, const T* residual, int64_t rows, int64_t in, int64_t out,
               int activation, T* y, void* saved, void* workspace, int64_t bytes, void* stream)
{
    if (int rc = check_shape(rows, in, out, activation))
        return rc;
    if (rows == 0 || out == 0)
        return MIQ_OK;
    MIQ_CHECK_ARG(y && (in == 0 || (x && w)), "null pointer");
    MIQ_CHECK_ARG(bytes >= workspace_bytes<T>(rows, in, out, activation, 0), "the workspace is too small");
    (void) workspace;
    int rc = MIQ_OK;
    with_activation(activation, [&](auto act) {
        rc = product<T, act.value>(x, in, 1, w, in, 1, rows, out, in, bias, residual, y, (Saved<T>*) saved,
                                   (hipStream_t) stream);
    });
    return rc;
}

template <typename T>
int linear_bwd(const T* g, const void* saved, const T* x, const T* w, int64_t rows, int64_t in, int64_t out,
               int activation, T* dx, T* dw, T* db, void* workspace, int64_t bytes, void* stream)
{
    if (int rc = check_shape(rows, in, out, activation))
        return rc;
    const bool kept = activation != MIQ_ACT_NONE;
    MIQ_CHECK_ARG(rows * out == 0 || (g && (saved || !kept)), "null pointer");
    MIQ_CHECK_ARG(rows * in == 0 || !dw || x, "dweight needs x");
    MIQ_CHECK_ARG(out * in == 0 || !dx || w, "dx needs weight");
    MIQ_CHECK_ARG(workspace && bytes >= workspace_bytes<T>(rows, in, out, activation, 1),
                  "the workspace is too small");
    hipStream_t s  = (hipStream_t) stream;
    const T* dz    = g;
    float* partial = (float*) ((char*) workspace + (kept ? up256(rows * out * (int64_t) sizeof(T)) : 0));
    if ((kept || db) && out > 0)
    {
        const int64_t slices = slope_slices(rows, out);
        const dim3 grid((unsigned) ((out + kBlock - 1) / kBlock), (unsigned) slices);
        with_activation(activation, [&](auto act) {
            hipLaunchKernelGGL((slope_kernel<T, act.value>), grid, dim3(kBlock), 0, s, g, (const Saved<T>*) saved,
                               rows, out, (rows + slices - 1) / slices, (T*) workspace, partial);
        });
        MIQ_CHECK_LAUNCH();
        if (kept)
            dz = (const T*) workspace;
        if (db)
            hipLaunchKernelGGL(join_columns_kernel<T>, dim3(grid.x), dim3(kBlock), 0, s, partial, slices, out, db);
        MIQ_CHECK_LAUNCH();
    }
    int rc = MIQ_OK;
    if (dx)
        rc = product<T, MIQ_ACT_NONE>(dz, out, 1, w, 1, in, rows, in, out, nullptr, nullptr, dx, nullptr, s);
    if (rc == MIQ_OK && dw)
        rc = product<T, MIQ_ACT_NONE>(dz, 1, out, x, 1, in, out, in, rows, nullptr, nullptr, dw, nullptr, s);
    return rc;
}
}   // namespace
}   // namespace miq

using namespace miq;

extern "C"
{
int64_t miq_linear_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int activation, int bf16,
                                   int backward)
{
    if (rows < 0 || in_features < 0 || out_features < 0)
        return 0;
    return bf16 ? workspace_bytes<uint16_t>(rows, in_features, out_features, activation, backward)
                : workspace_bytes<float>(rows, in_features, out_features, activation, backward);
}

int miq_linear_fwd_f32(const float* x, const float* weight, const float* bias, const float* residual, int64_t rows,
                       int64_t in_features, int64_t out_features, int activation, float* y, float* saved,
                       void* workspace, int64_t workspace_bytes, void* stream)
{
    return linear_fwd(x, weight, bias, residual, rows, in_features, out_features, activation, y, saved, workspace,
                      workspace_bytes, stream);
}

int miq_linear_fwd_bf16(const uint16_t* x, const uint16_t* weight, const uint16_t* bias, const uint16_t* residual,
                        int64_t rows, int64_t in_features, int64_t out_features, int activation, uint16_t* y,
                        uint16_t* saved, void* workspace, int64_t workspace_bytes, void* stream)
{
    return linear_fwd(x, weight, bias, residual, rows, in_features, out_features, activation, y, saved, workspace,
                      workspace_bytes, stream);
}

int miq_linear_bwd_f32(const float* grad, const float* saved, const float* x, const float* weight, int64_t rows,
                       int64_t in_features, int64_t out_features, int activation, float* dx, float* dweight,
                       float* dbias, void* workspace, int64_t workspace_bytes, void* stream)
{
    return linear_bwd(grad, saved, x, weight, rows, in_features, out_features, activation, dx, dweight, dbias,
                      workspace, workspace_bytes, stream);
}

int miq_linear_bwd_bf16(const uint16_t* grad, const uint16_t* saved, const uint16_t* x, const uint16_t* weight,
                        int64_t rows, int64_t in_features, int64_t out_features, int activation, uint16_t* dx,
                        uint16_t* dweight, uint16_t* dbias, void* workspace, int64_t workspace_bytes, void* stream)
{
    return linear_bwd(grad, saved, x, weight, rows, in_features, out_features, activation, dx, dweight, dbias,
                      workspace, workspace_bytes, stream);
}
}   // extern "C"
