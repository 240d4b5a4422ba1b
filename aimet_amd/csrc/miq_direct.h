// float32 products of middling size, straight from float32 operands: no pass over them beforehand.
//
// A float32 has 24 significant bits and is exactly the sum of three bfloat16 of 8 bits each, cut off one after the other:
//   p = x's upper half, q = (x - p)'s upper half, r = x - p - q
// all of x's sign, with x's exponent range (no scale is needed; of values under 2^-109 what is below bfloat16's smallest
// step, 2^-133, is lost).  With |q| < 2^-7 |x| and |r| < 2^-15 |x|.  Of the nine products of two such sums the six largest
// are formed on the matrix cores, smallest first; q r', r q' and r r' are less than 2^-21 of the product together, 2^-24.5 on
// average over normally distributed values.  What is left out has the product's sign: the result is that much nearer to zero.
// Operands are cut into parts on their way from LDS to the matrix unit.  That bounds it: on 128 x 128 tiles the
// vector unit is as busy with cutting (44 % of the time, by the counters) as the matrix unit with the six products (44 %),
// and the two hardly overlap.  [128, 4096] x [11008, 4096]^T: 77 us, the gradients 73 and 94; by halves 142, 237 and 160.
#ifndef MIQ_DIRECT_H
#define MIQ_DIRECT_H

#include "miq_product.h"

namespace miq
{
struct Parts
{
    s8v p, q, r;
};

__device__ __forceinline__ uint32_t upper_halves(float lo, float hi)
{
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

__device__ __forceinline__ Parts parts_of(const float* v)
{
    typedef uint32_t u4v __attribute__((ext_vector_type(4)));
    u4v p, q, r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float a = v[2 * i], b = v[2 * i + 1];
        const float a1 = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        const float b1 = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        const float a2 = a1 - __uint_as_float(__float_as_uint(a1) & 0xffff0000u);
        const float b2 = b1 - __uint_as_float(__float_as_uint(b1) & 0xffff0000u);
        p[i] = upper_halves(a, b);
        q[i] = upper_halves(a1, b1);
        r[i] = upper_halves(a2, b2);
    }
    return {__builtin_bit_cast(s8v, p), __builtin_bit_cast(s8v, q), __builtin_bit_cast(s8v, r)};
}

// What 8 values are to a sum that is not finite: bfloat16 that are NaN, infinite, zero or neither as they are, and of their
// sign.  (The upper half alone of a NaN may be an infinity, and that of the smallest values is zero.)
__device__ __forceinline__ s8v kinds_of(const float* v)
{
    s8v p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const uint32_t u = __float_as_uint(v[i]), m = u & 0x7fffffffu, sign = u >> 16 & 0x8000u;
        p[i] = (short) (m > 0x7f800000u ? 0x7fc0u : m != 0 && m < 0x00800000u ? sign | 0x0080u : u >> 16);
    }
    return p;
}

// 8 values of k (from 8 (lane / 16)) of row lane % 16 of a float32 slice of 32
template <bool COLUMNS, int CHUNKS>
struct DirectReader
{
    uint32_t at;
    __device__ __forceinline__ void place(int first, int lane)
    {
        if (!COLUMNS)
        {
            const int r = first + lane % 16;
            at          = r * 128 + exchanged<4>(r, lane / 16 * 2) * 16;
        }
        else
        {
            const int k = lane / 16 * 8, c = first + lane % 16;
            at          = k * (CHUNKS * 16) + exchanged<5>(k, c / 4) * 16 + c % 4 * 4;
        }
    }
    __device__ __forceinline__ void read(const char* lds, int i, float* v) const
    {
        if (!COLUMNS)
        {
            const char* from = lds + i * 2048;
            *(f4*) v         = *(const f4*) (from + at);
            *(f4*) (v + 4)   = *(const f4*) (from + (at ^ 16));
        }
        else
        {
            // 16 columns on are 4 chunks on: bits that are exchanged, and that the lane's part has from `first` alone
            const char* from = lds + (at ^ i * 64);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                v[u] = *(const float*) (from + u * (CHUNKS * 16));
        }
    }
};

struct DirectProduct
{
    Operand<float> a, b;
    int64_t k;
    int tiles_m, tiles_n, splits;
    float* partial;
    Epilogue<float> e;
};

template <int ACT, int WM, int WN, int FM, int FN, bool AC, bool BC>
__global__ __launch_bounds__(WM* WN * 64, 2) void direct_kernel(const DirectProduct p)
{
    constexpr int kWaves = WM * WN, kTM = WM * FM * 16, kTN = WN * FN * 16;
    using LA             = Loader<float, kTM, kWaves, AC, AC ? 5 : 4>;
    using LB             = Loader<float, kTN, kWaves, BC, BC ? 5 : 4>;
    constexpr int kDeep  = LA::kDeep;
    __shared__ __attribute__((aligned(1024))) char lds[2 * (LA::kBytes + LB::kBytes)];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int blocks = p.tiles_m * p.tiles_n;
    const int split  = blockIdx.x / blocks;
    int tm, tn;
    tile_of_block(blockIdx.x % blocks, blocks, p.tiles_m, p.tiles_n, &tm, &tn);
    const int64_t m0 = (int64_t) tm * kTM, n0 = (int64_t) tn * kTN;
    const int slices = (int) ((p.k + kDeep - 1) / kDeep);
    const int first = (int) ((int64_t) slices * split / p.splits), last = (int) ((int64_t) slices * (split + 1) / p.splits);

    DirectReader<AC, LA::kChunks> ra;
    DirectReader<BC, LB::kChunks> rb;
    ra.place(wm * FM * 16, lane);
    rb.place(wn * FN * 16, lane);

    f4 acc[FM][FN];
    const auto sum = [&](auto whole) {
        LA la;
        LB lb;
        la.start(p.a, m0, wave, lane);
        lb.start(p.b, n0, wave, lane);
        la.p += (int64_t) first * la.step;
        lb.p += (int64_t) first * lb.step;
        int64_t left     = p.k - (int64_t) first * kDeep;
        const auto issue = [&](int buffer) {
            const uint32_t to = lds_address(lds) + (uint32_t) buffer * (LA::kBytes + LB::kBytes);
            la.load(p.a, m0, to, wave, lane, left);
            lb.load(p.b, n0, to + LA::kBytes, wave, lane, left);
            left -= kDeep;
        };
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
        if (first < last)
            issue(0);
        for (int s = 0; s < last - first; ++s)
        {
            arrived();   // slice s has arrived, and everybody has read slice s - 1
            if (s + 1 < last - first)
                issue((s + 1) & 1);
            const char* sa = lds + (s & 1) * (LA::kBytes + LB::kBytes);
            const char* sb = sa + LA::kBytes;
            Parts fb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j)
            {
                float v[8];
                rb.read(sb, j, v);
                if constexpr (decltype(whole)::value)
                    fb[j] = parts_of(v);
                else
                    fb[j].p = kinds_of(v);
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
            {
                float v[8];
                ra.read(sa, i, v);
                Parts fa;
                constexpr auto kind = std::true_type();
                if constexpr (!decltype(whole)::value)
                    fa.p = kinds_of(v);
                else
                {
                    fa = parts_of(v);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = mfma_16x16x32(fb[j].p, fa.r, acc[i][j], kind);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = mfma_16x16x32(fb[j].r, fa.p, acc[i][j], kind);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = mfma_16x16x32(fb[j].q, fa.q, acc[i][j], kind);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = mfma_16x16x32(fb[j].p, fa.q, acc[i][j], kind);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = mfma_16x16x32(fb[j].q, fa.p, acc[i][j], kind);
                }
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = mfma_16x16x32(fb[j].p, fa.p, acc[i][j], kind);
            }
        }
    };
    sum(std::true_type());

    // An infinity or a NaN has no parts beyond the first: where the sum is not finite, it is formed again of kinds_of(), which
    // makes of it what float32 arithmetic would.  (If that is finite the sum has left float32's range, and stays what it is.)
    bool finite = true;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                finite = finite && __builtin_isfinite(acc[i][j][u]);
    if (__syncthreads_or(!finite))
    {
        f4 kept[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                kept[i][j] = acc[i][j];
        sum(std::false_type());
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    acc[i][j][u] = __builtin_isfinite(kept[i][j][u]) || __builtin_isfinite(acc[i][j][u])
                                       ? kept[i][j][u]
                                       : acc[i][j][u];
    }

#pragma unroll
    for (int i = 0; i < FM; ++i)
    {
        const int64_t r = m0 + wm * FM * 16 + i * 16 + lane % 16;
        if (r >= p.e.m)
            continue;
#pragma unroll
        for (int j = 0; j < FN; ++j)
        {
            const int64_t q = n0 + wn * FN * 16 + j * 16 + lane / 16 * 4;
            if (q >= p.e.n)
                continue;
            float z[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            if (p.splits == 1)
                finish4<ACT>(p.e, r, q, z);
            else
                store4(p.partial + ((int64_t) split * p.e.m + r) * p.e.n + q, p.e.n - q, z);
        }
    }
}
}   // namespace miq

#endif
