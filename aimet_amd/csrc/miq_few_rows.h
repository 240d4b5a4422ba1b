// Products with few rows on the left (single tokens, small batches): the weight is read once, from memory to registers,
// and nothing else takes time.  [1, 4096] x [11008, 4096]^T bfloat16: 18.3 us (4.9 TB/s); [16, 4096] x [4096, 4096]^T
// float32: 18 us (3.8 TB/s), its input's gradient 20.  The 128 x 128 tiles take 21.6 us for the first and, with the halves
// they need, 82 for the second.  From 17 rows on the tiles (bfloat16) and the direct products (float32) are faster.
#ifndef MIQ_FEW_ROWS_H
#define MIQ_FEW_ROWS_H

#include "miq_product.h"

namespace miq
{
__device__ __forceinline__ void load4(const float* p, float* v)
{
    load_any(p, v);
}
__device__ __forceinline__ void load4(const uint16_t* p, float* v)
{
    typedef unsigned short any_s4 __attribute__((ext_vector_type(4), aligned(2)));
    const any_s4 w = *(const any_s4*) p;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = bf16_to_f32(w[i]);
}

// 16 bytes of a row (8 or 4 values of k) in the form the matrix unit takes them
template <typename T>
struct Chunk;

template <>
struct Chunk<uint16_t>
{
    static constexpr int VEC = 8;
    s8v v;
    __device__ __forceinline__ void load(const uint16_t* p)
    {
        typedef short any_s8 __attribute__((ext_vector_type(8), aligned(2)));
        v = *(const any_s8*) p;
    }
    __device__ __forceinline__ void load_some(const uint16_t* p, int64_t left)
    {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            v[i] = i < left ? (short) p[i] : (short) 0;
    }
    static __device__ __forceinline__ f4 mad(const Chunk& n, const Chunk& m, f4 c)
    {
        return mfma_16x16x32(n.v, m.v, c, std::true_type());
    }
};

// float32 at full precision: four v_mfma_f32_16x16x4, each with one value of the chunk a lane
template <>
struct Chunk<float>
{
    static constexpr int VEC = 4;
    f4 v;
    __device__ __forceinline__ void load(const float* p)
    {
        v = *(const any_f4*) p;
    }
    __device__ __forceinline__ void load_some(const float* p, int64_t left)
    {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            v[i] = i < left ? p[i] : 0.f;
    }
    static __device__ __forceinline__ f4 mad(const Chunk& n, const Chunk& m, f4 c)
    {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(n.v[i], m.v[i], c, 0, 0, 0);
        return c;
    }
};

// C[m, n] = act(sum over k of a[m][k] b[n][k] + bias) + residual for up to 16 rows of a.
// A block makes 16 columns; its waves share the sum over k and add their parts through LDS, in order.  A wave takes
// 16 rows of b at a time, 64 bytes of each: lane l row l % 16, bytes from 16 (l / 16).  Rows of a and b past the end
// are the last one again: what they make is not stored.
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void few_rows_kernel(const T* __restrict__ a, const T* __restrict__ b, int64_t k,
                                                        const Epilogue<T> e)
{
    using C             = Chunk<T>;
    constexpr int kStep = 4 * C::VEC, kUnroll = 8;
    extern __shared__ f4 parts[];   // [waves][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
              waves = blockDim.x >> 6;
    const int64_t n0    = (int64_t) blockIdx.x * 16;
    const int64_t whole = k / kStep, first = whole * wave / waves, last = whole * (wave + 1) / waves;
    const int in    = lane / 16 * C::VEC;
    const int64_t n = n0 + lane % 16, m = lane % 16;
    const T* pb     = b + (n < e.n ? n : e.n - 1) * k + first * kStep + in;
    const T* pa     = a + (m < e.m ? m : e.m - 1) * k + first * kStep + in;
    f4 acc          = f4{0.f, 0.f, 0.f, 0.f};
    int64_t s       = first;
    for (; s + kUnroll <= last; s += kUnroll)
    {
        C wide[kUnroll], rows[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            wide[u].load(pb + u * kStep);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            rows[u].load(pa + u * kStep);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            acc = C::mad(wide[u], rows[u], acc);
        pb += kUnroll * kStep;
        pa += kUnroll * kStep;
    }
    const int64_t end = last + (wave == waves - 1 && whole * kStep < k ? 1 : 0);
    for (; s < end; ++s)
    {
        const int64_t left = k - s * kStep - in;
        C fa, fb;
        if (left >= C::VEC)
        {
            fb.load(pb);
            fa.load(pa);
        }
        else
        {
            fb.load_some(pb, left);
            fa.load_some(pa, left);
        }
        pb += kStep;
        pa += kStep;
        acc = C::mad(fb, fa, acc);
    }
    parts[threadIdx.x] = acc;
    __syncthreads();
    if (threadIdx.x >= 64)
        return;
    for (int w = 1; w < waves; ++w)
        acc += parts[w * 64 + lane];
    if (m < e.m)
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (n0 + lane / 16 * 4 + u < e.n)
                finish1<T, ACT>(e, m, n0 + lane / 16 * 4 + u, acc[u]);
}

// C[m, n] or, for one of several pieces of k, partial[split][m][n] = sum over k of a[m][k] b[k][n], up to 16 rows of a.
// b is read as it lies: lane l takes 16 bytes, VEC columns from VEC (l % 16), of row 4 (l / 16) + t of 16 rows, t = 0 .. 3.
// As float32 they are the first factor of v_mfma_f32_16x16x4: value u of all lanes makes columns VEC r + u, r = 0 .. 15,
// so that a lane ends up with 4 VEC consecutive columns of one m.  A block makes 16 VEC columns; its waves share the sum.
template <typename T>
__global__ __launch_bounds__(512) void few_rows_columns_kernel(const T* __restrict__ a, int64_t lda,
                                                               const T* __restrict__ b, int64_t k, int64_t per_split,
                                                               float* __restrict__ partial, const Epilogue<T> e)
{
    constexpr int VEC = IOTraits<T>::VEC, kUnroll = 2;
    extern __shared__ f4 parts[];   // [waves][VEC][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
              waves = blockDim.x >> 6;
    const int64_t c    = ((int64_t) blockIdx.x * 16 + lane % 16) * VEC;
    const int64_t from = blockIdx.y * per_split, to = from + per_split < k ? from + per_split : k;
    const int64_t steps = to > from ? (to - from + 15) / 16 : 0;
    const int64_t first = steps * wave / waves, last = steps * (wave + 1) / waves;
    const T* pa       = a + (lane % 16 < e.m ? lane % 16 : e.m - 1) * lda;
    const bool inside = c + VEC <= e.n;
    f4 acc[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u)
        acc[u] = f4{0.f, 0.f, 0.f, 0.f};
    for (int64_t s = first; s < last; s += kUnroll)
    {
        float w[kUnroll][4][VEC], x[kUnroll][4];
#pragma unroll
        for (int v = 0; v < kUnroll; ++v)
        {
            const int64_t k0   = from + (s + v) * 16 + lane / 16 * 4;
            const int64_t left = s + v < last ? to - k0 : 0;
            const bool whole   = left >= 4;
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (whole && inside)
                    load_any(b + (k0 + t) * e.n + c, w[v][t]);
                else
#pragma unroll
                    for (int u = 0; u < VEC; ++u)
                        w[v][t][u] = t < left && c + u < e.n ? value_at(b + (k0 + t) * e.n + c + u) : 0.f;
            if (whole)
                load4(pa + k0, x[v]);
            else
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    x[v][t] = t < left ? value_at(pa + k0 + t) : 0.f;
        }
#pragma unroll
        for (int v = 0; v < kUnroll; ++v)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int u = 0; u < VEC; ++u)
                    acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[v][t][u], x[v][t], acc[u], 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < VEC; ++u)
        parts[(wave * VEC + u) * 64 + lane] = acc[u];
    __syncthreads();
    // a thread finishes 4 VEC values, VEC at a time: row l % 16, value v of lane l
    for (int at = threadIdx.x; at < 64 * 4; at += blockDim.x)
    {
        const int v = at % 4, l = at / 4;
        const int64_t row = l % 16, q = ((int64_t) blockIdx.x * 16 + l / 16 * 4 + v) * VEC;
        if (row >= e.m)
            continue;
#pragma unroll
        for (int u = 0; u < VEC; ++u)
        {
            float z = 0.f;
            for (int w = 0; w < waves; ++w)
                z += parts[(w * VEC + u) * 64 + l][v];
            if (q + u >= e.n)
                continue;
            if (partial)
                partial[((int64_t) blockIdx.y * e.m + row) * e.n + q + u] = z;
            else
                finish1<T, MIQ_ACT_NONE>(e, row, q + u, z);
        }
    }
}

// C[m, n] = sum over k of a[k][m] b[k][n] for a short k (the weight's gradient of a small batch), float32: writing C is
// all that counts.  A wave makes 64 x 64 values from operands read straight from the caches.
__global__ __launch_bounds__(kBlock) void short_sum_kernel(const float* __restrict__ a, int64_t lda,
                                                           const float* __restrict__ b, int k, const Epilogue<float> e)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tiles_n = (e.n + 127) / 128;
    const int64_t m0 = blockIdx.x / tiles_n * 128 + wave / 2 * 64, n0 = blockIdx.x % tiles_n * 128 + wave % 2 * 64;
    f4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < k; k0 += 4)
    {
        const int kk = k0 + lane / 16;
        float fa[4], fb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const int64_t m = m0 + i * 16 + lane % 16, n = n0 + i * 16 + lane % 16;
            fa[i] = kk < k && m < e.m ? a[kk * lda + m] : 0.f;
            fb[i] = kk < k && n < e.n ? b[kk * e.n + n] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j], fa[i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const int64_t m = m0 + i * 16 + lane % 16;
        if (m >= e.m)
            continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const int64_t n = n0 + j * 16 + lane / 16 * 4;
            const float z[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            if (n + 4 <= e.n)
                store_any(e.c + m * e.n + n, z);
            else
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (n + u < e.n)
                        e.c[m * e.n + n + u] = z[u];
        }
    }
}
}   // namespace miq

#endif
