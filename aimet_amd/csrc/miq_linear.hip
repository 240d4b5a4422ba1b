// Matrix product with bias, activation and residual in its epilogue, and its backward pass, for gfx950.
//
//   z = x w^T + b, y = act(z) + residual                          x [rows, in], w [out, in], y [rows, out]
//   dz = g act'(z), dx = dz w, dw = dz^T x, db = sum over rows of dz, dresidual = g
#include "miq_direct.h"
#include "miq_few_rows.h"
#include "miq_halves.h"

#include <algorithm>

namespace miq
{
namespace
{
// ------------------------------------------------------------------------------------------ operands made ready
// Tiles read whole 16-byte chunks.  Tensors whose rows are whole chunks are read as they lie; others are copied, with
// zeros behind their rows.
//
// float32 operands of large products become two halves of 11 significant bits each, row by row (a row: what shares one m
// or n):
//   s = 14 - floor(log2 of the row's largest finite magnitude), t = x 2^s, coarse = half(t), fine = half(t - coarse)
// so |t - coarse - fine| <= 2^-23 |t| as long as fine is a normal half, and never more than 2^-25, which is 2^-39 of the
// row's largest.  A product of two operands is the sum of coarse coarse + coarse fine + fine coarse; fine fine, which is
// left out, is at most 2^-22 of it and has no sign of its own: about the error of float32 arithmetic itself.  Three
// products in the half-precision matrix unit take a fifth of the time of one in the float32 one.
// coarse of an infinity or NaN is itself, its fine is 0.
//
// A value below 2^-17 of its row's largest loses bits, and one below 2^-39 is lost.  Where the row's large values meet zeros,
// that is all there is of the sum.  So each row carries how many of its values lost bits ("lost"; of a row of zeros -2^30,
// since its sums are zeros whatever the other operand lost), and halves_kernel forms again, from float32 operands, the
// sums that this may have changed by more than float32 arithmetic would.
__device__ __forceinline__ int row_shift(uint32_t largest /* bits of a finite float32 */)
{
    if (largest == 0)
        return 0;
    const int e = (int) (largest >> 23);
    return 14 - (e ? e - 127 : (31 - __clz(largest)) - 149);
}

// whether bits of x were lost
__device__ __forceinline__ bool split_value(float x, int shift, uint16_t* coarse, uint16_t* fine)
{
    const float t    = ldexpf(x, shift);
    const _Float16 c = (_Float16) t;
    const float f    = t - (float) c;
    const _Float16 d = __builtin_isfinite(t) ? (_Float16) f : (_Float16) 0.f;
    *coarse          = __builtin_bit_cast(uint16_t, c);
    *fine            = __builtin_bit_cast(uint16_t, d);
    return fabsf(f - (float) d) > 0x1p-22f * fabsf(t) || (t == 0.f && x != 0.f);
}

__device__ __forceinline__ uint32_t finite_magnitude(float x)
{
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// 8 values as 16-bit operands; how many of them lost bits
__device__ __forceinline__ int put_parts(const float* v, int shift, uint16_t* coarse, uint16_t* fine)
{
    uint16_t c[8], f[8];
    int lost = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
        lost += split_value(v[u], shift, c + u, f + u);
    *(uint4*) coarse = make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16);
    *(uint4*) fine   = make_uint4(f[0] | f[1] << 16, f[2] | f[3] << 16, f[4] | f[5] << 16, f[6] | f[7] << 16);
    return lost;
}
// out[r] = the halves of src[r][0 .. k), of zeros up to kp (a multiple of kHalves): for every kHalves values their coarse
// halves and then their fine ones; scale[r] = -s, lost[r] as above.
// LANES threads hold a row of up to 32 LANES values in registers between its largest value and its halves; of a longer
// one what is past them is read again.
template <int LANES>
__global__ __launch_bounds__(kBlock) void pack_rows_kernel(const float* __restrict__ src, int64_t ld, int64_t rows,
                                                           int64_t k, int64_t kp, uint16_t* __restrict__ out,
                                                           int* __restrict__ scale, int* __restrict__ lost)
{
    constexpr int kHeld = 4;
    const int lane  = threadIdx.x % LANES;
    const int64_t r = block_index() * (kBlock / LANES) + threadIdx.x / LANES;
    if (r >= rows)
        return;
    const float* from = src + r * ld;
    float v[kHeld][8], t[8];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        load8(from + (i * LANES + lane) * 8, k - (i * LANES + lane) * 8, v[i]);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
#pragma unroll
        for (int u = 0; u < 8; ++u)
            largest = max(largest, finite_magnitude(v[i][u]));
    for (int64_t c = (kHeld * LANES + lane) * 8; c < k; c += LANES * 8)
    {
        load8(from + c, k - c, t);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            largest = max(largest, finite_magnitude(t[u]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        largest = max(largest, (uint32_t) __shfl_xor((int) largest, o, 64));
    if constexpr (LANES > 64)
    {
        __shared__ uint32_t lds[LANES / 64];
        if ((threadIdx.x & 63) == 0)
            lds[threadIdx.x >> 6] = largest;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LANES / 64; ++i)
            largest = max(largest, lds[i]);
    }
    const int shift = row_shift(largest);
    uint16_t* to    = out + r * 2 * kp;
    int without     = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
    {
        const int64_t c = (i * LANES + lane) * 8;
        if (c < kp)
            without += put_parts(v[i], shift, to + place_of_half(c), to + place_of_half(c) + kHalves);
    }
    for (int64_t c = (kHeld * LANES + lane) * 8; c < kp; c += LANES * 8)
    {
        load8(from + c, k - c, t);
        without += put_parts(t, shift, to + place_of_half(c), to + place_of_half(c) + kHalves);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        without += __shfl_xor(without, o, 64);
    if constexpr (LANES > 64)
    {
        __shared__ int lds[LANES / 64];
        if ((threadIdx.x & 63) == 0)
            lds[threadIdx.x >> 6] = without;
        __syncthreads();
        without = 0;
#pragma unroll
        for (int i = 0; i < LANES / 64; ++i)
            without += lds[i];
    }
    if (lane == 0)
    {
        scale[r] = -shift;
        lost[r]  = largest ? without : kZeroRow;
    }
}

// out[r][0 .. kp) = src[r][0 .. k), zeros behind
template <typename T>
__global__ __launch_bounds__(kBlock) void copy_rows_kernel(const T* __restrict__ src, int64_t rows, int64_t k,
                                                           int64_t kp, T* __restrict__ out)
{
    constexpr int VEC = IOTraits<T>::VEC;
    const int64_t per = kp / VEC, at = block_index() * kBlock + threadIdx.x;
    if (at >= rows * per)
        return;
    const int64_t r = at / per, c = at % per * VEC;
    any_u4 v          = {0u, 0u, 0u, 0u};
    if (c + VEC <= k)
        v = *(const any_u4*) (src + r * k + c);
    else
#pragma unroll
        for (int u = 0; u < VEC; ++u)
            if (c + u < k)
            {
                if constexpr (VEC == 4)
                    v[u] = __float_as_uint(src[r * k + c + u]);
                else
                    v[u / 2] |= (uint32_t) src[r * k + c + u] << (u % 2 * 16);
            }
    *(uint4*) (out + r * kp + c) = make_uint4(v[0], v[1], v[2], v[3]);
}

// largest[slice][c] = largest finite magnitude (its bits) in a slice of the rows of column c of src [k][count]: 64 threads
// of 4 columns across, 4 rows at a time.  lost[c] = 0, for pack_columns_kernel to add to.
__global__ __launch_bounds__(kBlock) void column_max_kernel(const float* __restrict__ src, int64_t ld, int64_t k, int64_t count,
                                                            int64_t rows_per_slice, uint32_t* __restrict__ largest,
                                                            int* __restrict__ lost)
{
    __shared__ uint32_t lds[4][256];
    const int across    = threadIdx.x % 64, down = threadIdx.x / 64;
    const int64_t c     = ((int64_t) blockIdx.x * 64 + across) * 4;
    const int64_t first = blockIdx.y * rows_per_slice;
    const int64_t last  = first + rows_per_slice < k ? first + rows_per_slice : k;
    uint32_t m[4]       = {};
    if (c + 4 <= count)
    {
#pragma unroll 4
        for (int64_t r = first + down; r < last; r += 4)
        {
            float v[4];
            load_any(src + r * ld + c, v);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                m[u] = max(m[u], finite_magnitude(v[u]));
        }
    }
    else
        for (int64_t r = first + down; r < last; r += 4)
            for (int u = 0; u < 4; ++u)
                if (c + u < count)
                    m[u] = max(m[u], finite_magnitude(src[r * ld + c + u]));
#pragma unroll
    for (int u = 0; u < 4; ++u)
        lds[down][u * 64 + across] = m[u];
    __syncthreads();
    const int at = threadIdx.x % 4 * 64 + threadIdx.x / 4;   // column threadIdx.x of the block's 256
    const int64_t q = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (q >= count)
        return;
    largest[blockIdx.y * count + q] = max(max(lds[0][at], lds[1][at]), max(lds[2][at], lds[3][at]));
    if (blockIdx.y == 0)
        lost[q] = 0;
}

// As pack_rows_kernel, of the transpose: src [k][count], row r of the result is column r of src.  64 x 64 values a block,
// through LDS.
__global__ __launch_bounds__(kBlock) void pack_columns_kernel(const float* __restrict__ src, int64_t ld, int64_t k,
                                                              int64_t count, int64_t kp,
                                                              const uint32_t* __restrict__ largest, int slices,
                                                              uint16_t* __restrict__ out, int* __restrict__ scale,
                                                              int* __restrict__ lost)
{
    __shared__ float tile[64][65];
    __shared__ int shifts[64], without[64];
    const int64_t across = (count + 63) / 64;
    const int64_t r0 = blockIdx.x % across * 64, k0 = blockIdx.x / across * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        const int64_t kk = k0 + i * 4 + wave;
        tile[i * 4 + wave][lane] = kk < k && r0 + lane < count ? src[kk * ld + r0 + lane] : 0.f;
    }
    if (threadIdx.x < 64)
    {
        uint32_t m = 0;
        if (r0 + lane < count)
            for (int i = 0; i < slices; ++i)
                m = max(m, largest[i * count + r0 + lane]);
        shifts[lane]  = row_shift(m);
        without[lane] = k0 == 0 && m == 0 ? kZeroRow : 0;
        if (k0 == 0 && r0 + lane < count)
            scale[r0 + lane] = -row_shift(m);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
    {
        const int r = (i * kBlock + threadIdx.x) / 8, c = threadIdx.x % 8 * 8;
        if (r0 + r >= count || k0 + c >= kp)
            continue;
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            v[u] = tile[c + u][r];
        uint16_t* to = out + (r0 + r) * 2 * kp + place_of_half(k0 + c);
        if (const int n = put_parts(v, shifts[r], to, to + kHalves))
            atomicAdd(&without[r], n);
    }
    __syncthreads();
    // (few columns lose anything; whole numbers have one sum in any order)
    if (threadIdx.x < 64 && r0 + lane < count && without[lane])
        atomicAdd(lost + r0 + lane, without[lane]);
}

// dz = g act'(z) and its column sums over a slice of the rows, at memory's rate (4096 x 11008 bfloat16: 65 us, 4.2 TB/s;
// 4096 x 4096 float32: 41 us, 4.9 TB/s): a thread takes 8 columns, 32 threads across and 8 rows at
// a time.  dz may be null for ACT none; its rows are `ld` values apart, zeros behind the last column.
// For bfloat16 tensors dz is rounded to bfloat16 here (the column sums are of what it was before), for it is a factor of two
// products whose matrix instructions take nothing wider beside a bfloat16: in two parts, it would double them, 590 us more on
// 4096 x 4096 -> 11008.  The gradients behind an activation are then off by 0.0024 of their norm instead of the 0.0017 that
// their own rounding makes.
template <typename T, int ACT>
__global__ __launch_bounds__(kBlock) void slope_kernel(const T* __restrict__ g, const Saved<T>* __restrict__ z,
                                                       int64_t rows, int64_t cols, int64_t ld, int64_t rows_per_slice,
                                                       T* __restrict__ dz, float* __restrict__ partial)
{
    constexpr int VEC = 8, kAcross = 32, kDown = kBlock / kAcross;
    __shared__ float lds[kDown][kAcross * VEC];
    const int across = threadIdx.x % kAcross, down = threadIdx.x / kAcross;
    const int64_t c     = ((int64_t) blockIdx.x * kAcross + across) * VEC;
    const int64_t first = blockIdx.y * rows_per_slice;
    const int64_t last  = first + rows_per_slice < rows ? first + rows_per_slice : rows;
    float sum[VEC]      = {};
    if (c < cols)
#pragma unroll 2
        for (int64_t r = first + down; r < last; r += kDown)
        {
            const int64_t at = r * cols + c;
            float d[VEC], s[VEC];
            load8(g + at, cols - c, d);
            if constexpr (ACT != MIQ_ACT_NONE)
            {
                load8(z + at, cols - c, s);
#pragma unroll
                for (int u = 0; u < VEC; ++u)
                    d[u] *= act_slope<ACT>(s[u]);
            }
            if (dz)
                store8(dz + r * ld + c, ld - c, d);
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                sum[u] += d[u];
        }
    if (!partial)
        return;
#pragma unroll
    for (int u = 0; u < VEC; ++u)
        lds[down][across * VEC + u] = sum[u];
    __syncthreads();
    for (int i = threadIdx.x; i < kAcross * VEC; i += kBlock)
    {
        const int64_t q = (int64_t) blockIdx.x * kAcross * VEC + i;
        if (q >= cols)
            continue;
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < kDown; ++k)
            t += lds[k][i];
        partial[(int64_t) blockIdx.y * cols + q] = t;
    }
}

// adds the slices' sums: 64 columns a block, 4 threads a column
template <typename T>
__global__ __launch_bounds__(kBlock) void join_columns_kernel(const float* __restrict__ partial, int64_t slices,
                                                              int64_t cols, T* __restrict__ out)
{
    __shared__ float lds[4][64];
    const int64_t c = (int64_t) blockIdx.x * 64 + threadIdx.x % 64;
    const int part  = threadIdx.x / 64;
    float s         = 0.f;
    if (c < cols)
        for (int64_t k = part; k < slices; k += 4)
            s += partial[k * cols + c];
    lds[part][threadIdx.x % 64] = s;
    __syncthreads();
    if (part == 0 && c < cols)
        IOTraits<T>::store1(out + c, (lds[0][threadIdx.x] + lds[1][threadIdx.x]) +
                                         (lds[2][threadIdx.x] + lds[3][threadIdx.x]));
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
    const int64_t columns = std::max<int64_t>(1, (cols + kBlock - 1) / kBlock);   // (a layer may have no outputs)
    return std::max<int64_t>(1, std::min<int64_t>((1024 + columns - 1) / columns, rows / 16));
}

int64_t up256(int64_t n)
{
    return (n + 255) / 256 * 256;
}

// Longest row of an operand, in values of up to 4 bytes (a value's two halves take 4): a load spans 8 rows, and a lane's
// offset within them has 32 bits
constexpr int64_t kLongest = 1 << 27;

int check_shape(int64_t rows, int64_t in, int64_t out, int activation)
{
    MIQ_CHECK_ARG(rows >= 0 && in >= 0 && out >= 0, "rows, in_features and out_features must not be negative");
    MIQ_CHECK_ARG(rows <= INT32_MAX, "rows must be below 2^31");
    MIQ_CHECK_ARG(in <= kLongest && out <= kLongest, "in_features and out_features must be at most 2^27");
    MIQ_CHECK_ARG(activation >= MIQ_ACT_NONE && activation <= MIQ_ACT_GELU_TANH, "unknown activation %d", activation);
    return MIQ_OK;
}

// ------------------------------------------------------------------------------------------------ host side
bool aligned(const void* p)
{
    return ((uintptr_t) p & 15) == 0;
}

// A matrix that a product reads: k contiguous ("rows", [count][k]) or count contiguous ("columns", [k][count])
template <typename T>
struct Matrix
{
    const T* p;
    int64_t count, k;
    bool columns;
    bool at16;    // p is a multiple of 16 bytes
    int64_t ld;   // values from one row of memory to the next; what is past a row's end is zeros, if anything

    int64_t inner() const
    {
        return columns ? count : k;
    }
    int64_t outer() const
    {
        return columns ? k : count;
    }
    bool whole() const   // every row is whole 16-byte chunks
    {
        return at16 && ld * (int64_t) sizeof(T) % 16 == 0;
    }
};

// rows of whole 16-byte chunks
template <typename T>
int64_t padded(int64_t n)
{
    constexpr int VEC = 16 / sizeof(T);
    return (n + VEC - 1) / VEC * VEC;
}

int64_t max_slices(int64_t k)
{
    return std::max<int64_t>(1, std::min<int64_t>(32, k / 16));
}

// Whether a float32 product is formed from its operands as they lie (miq_direct.h) or from halves made beforehand
// (miq_halves.h).  The first runs at about 160 TFLOP/s (130 on columns, whole tiles counted), the second at up to 450 once the halves are there; making them takes
// 2 ps a value of an operand in rows and 3 ps in columns (one more pass), and 18 us of launches, 15 more for each operand
// in columns.  The rule is within 5 % of the better way on most of 90 measured products.  In us, as they lie and by halves:
// [256, 4096] x [4096, 4096]^T 62 and 71, [512, 4096] x [4096, 4096]^T 106 and 93, the input's gradient of
// [512, 4096] x [11008, 4096]^T 246 and 263, of [768, 4096] x [4096, 4096]^T 172 and 141, the weight's gradient of
// [512, 4096] x [4096, 4096]^T 102 and 91.
// Sums too long for rows of halves (a weight's gradient over more rows than that: both operands in columns) take the first.
template <typename T>
bool direct_pays(const Matrix<T>& a, const Matrix<T>& b)
{
    if (a.k > kLongest)
        return true;
    const auto halves = [](const Matrix<T>& x, double columns) {
        return (double) x.count * x.k * (x.columns ? columns : 2e-12) + (x.columns ? 15e-6 : 0);
    };
    const auto tiles = [](int64_t n) { return (double) ((n + 127) / 128 * 128); };
    return (a.columns ? 4.2e-15 : 3.5e-15) * 2.0 * tiles(a.count) * tiles(b.count) * a.k <=
           18e-6 + halves(a, 2.5e-12) + halves(b, 3e-12);
}

enum class Way
{
    kFewRows,      // few rows: b is read as it lies, by the kernels of miq_few_rows.h
    kFewColumns,   // the same, b in columns
    kShortSum,     // float32, both in columns, k short
    kDirect,       // float32, from the operands as they lie
    kTiles         // 16-bit operands
};

struct Plan
{
    Way way;
    int64_t kp;   // kTiles, float32: length of the rows of halves
    bool big;     // kTiles: 256 x 256, else 128 x 128; kDirect: 128 x 128, else 64 x 128
    int splits;
    int64_t a_bytes, b_bytes, scale_a, scale_b, partial, total;   // of the workspace (scale: scale, lost, columns' maxima)
};

// Tiles and pieces of the sum for a product of `slices` slices a pass whose values take `bytes`.  What a launch costs, in
// us, as measured on many shapes (within 10 % for most that are whole tiles and slices; others, whose loads are guarded, take up to
// twice as long: 30 instead of 16 for [1021, 1003] x [1531, 1003]^T): 5, and for each round of tiles that the device holds at a time
//   256 x 256, one a CU: 1.5 a slice, 1.25 when half of the CUs have none, and the result at 20 bytes a ns and CU
//   128 x 128, two a CU: 1.05 a slice, 0.6 when there is one, and half of that, for one writes while the other sums
// and to join the pieces 4 and 1 for each million of partial values.  E.g. bfloat16 [4096, 1024] x [1024, 1024]^T: 15 whole,
// 26 in two pieces; [512, 4096] x [4096, 4096]^T: 42, 32 and 32 in two and four; [2048, 11008] x [4096, 11008]^T: 191 in
// 128 x 128 tiles, 165 in 256 x 256 in two pieces.
void choose_tiles(int64_t m, int64_t n, int64_t slices, int passes, int bytes, Plan* p)
{
    double best = 1e30;
    for (const bool big : {false, true})
    {
        const int64_t side = big ? 256 : 128, tiles = (m + side - 1) / side * ((n + side - 1) / side);
        for (int64_t splits = 1; splits <= 32 && (splits == 1 || slices >= 4 * splits); splits *= 2)
        {
            const int64_t blocks = tiles * splits, at_once = big ? 256 : 512, rounds = (blocks + at_once - 1) / at_once;
            const bool sparse    = rounds == 1 && blocks <= at_once / 2;
            const double slice   = big ? (sparse ? 1.25 : 1.5) : (sparse ? 0.6 : 1.05);
            const double write   = (big ? 1.0 : 0.25) * 256 * 256 * bytes / 20e3;
            const double cost    = 5 + (double) rounds * (((slices + splits - 1) / splits) * passes * slice + write) +
                                (splits > 1 ? 4 + 1e-6 * splits * m * n : 0);
            if (cost < best)
            {
                best      = cost;
                p->big    = big;
                p->splits = (int) splits;
            }
        }
    }
}

template <typename T>
Plan plan_product(const Matrix<T>& a, const Matrix<T>& b)
{
    constexpr bool kF32 = std::is_same<T, float>::value;
    Plan p              = {};
    p.splits            = 1;
    const int64_t m = a.count, n = b.count, k = a.k;
    const auto done = [&] {
        p.partial = p.splits > 1 ? up256(p.splits * m * n * 4) : 0;
        p.total   = p.a_bytes + p.b_bytes + p.scale_a + p.scale_b + p.partial;
        return p;
    };
    // rows that are not whole chunks are copied, with zeros behind them
    const auto copied = [&](const Matrix<T>& x) {
        return x.whole() ? 0 : up256(x.outer() * padded<T>(x.inner()) * (int64_t) sizeof(T));
    };
    const auto tiles = [&](int64_t tm, int64_t tn) { return (m + tm - 1) / tm * ((n + tn - 1) / tn); };
    if (!a.columns && !b.columns && m <= 16)
    {
        p.way = Way::kFewRows;
        return done();
    }
    // (by the row's length, not by where b starts: a sum's order is the same wherever its operands lie)
    if (!a.columns && b.columns && m <= 16 && (kF32 || padded<T>(b.ld) != b.ld))
    {
        // about 2048 waves in blocks of 8; pieces of k of 128 at least
        const int64_t wide = (n + 16 * IOTraits<T>::VEC - 1) / (16 * IOTraits<T>::VEC);
        p.way    = Way::kFewColumns;
        p.splits = (int) std::max<int64_t>(1, std::min<int64_t>(256 / std::max<int64_t>(wide, 1), k / 128));
        return done();
    }
    if (kF32 && a.columns && b.columns && k <= 16)
    {
        p.way = Way::kShortSum;
        return done();
    }
    if (kF32 && direct_pays(a, b))
    {
        p.way = Way::kDirect;
        p.a_bytes = copied(a), p.b_bytes = copied(b);
        p.big = m > 64;
        p.splits = (int) std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(tiles(p.big ? 128 : 64, 128), 1), k / 256));
        return done();
    }
    p.way = Way::kTiles;
    choose_tiles(m, n, (k + kSlice - 1) / kSlice, kF32 ? 3 : 1, (int) sizeof(T), &p);
    p.a_bytes = copied(a), p.b_bytes = copied(b);
    if (kF32)
    {
        p.kp      = (k + kHalves - 1) / kHalves * kHalves;
        p.a_bytes = up256(m * 2 * p.kp * 2), p.b_bytes = up256(n * 2 * p.kp * 2);
        p.scale_a = up256(m * 4 * (2 + (a.columns ? max_slices(k) : 0)));
        p.scale_b = up256(n * 4 * (2 + (b.columns ? max_slices(k) : 0)));
    }
    return done();
}

template <typename T>
int copy_rows(const T* src, int64_t rows, int64_t k, int64_t kp, T* to, hipStream_t s)
{
    const int64_t blocks = (rows * (kp / IOTraits<T>::VEC) + kBlock - 1) / kBlock;
    if (blocks == 0)
        return MIQ_OK;
    hipLaunchKernelGGL(copy_rows_kernel<T>, grid_of(blocks, kBlock), dim3(kBlock), 0, s, src, rows, k, kp, to);
    MIQ_CHECK_LAUNCH();
    return MIQ_OK;
}

int pack(const Matrix<float>& x, int64_t kp, char* to, char* scale, hipStream_t s)
{
    if (x.count == 0 || kp == 0)
        return MIQ_OK;
    int* exponents    = (int*) scale;
    int* lost         = exponents + x.count;
    uint32_t* largest = (uint32_t*) lost + x.count;
    if (!x.columns)
    {
        if (x.k <= 2048)
            hipLaunchKernelGGL(pack_rows_kernel<64>, grid_of((x.count + 3) / 4, kBlock), dim3(kBlock), 0, s, x.p, x.ld,
                               x.count, x.k, kp, (uint16_t*) to, exponents, lost);
        else
            hipLaunchKernelGGL(pack_rows_kernel<256>, grid_of(x.count, kBlock), dim3(kBlock), 0, s, x.p, x.ld, x.count,
                               x.k, kp, (uint16_t*) to, exponents, lost);
        MIQ_CHECK_LAUNCH();
        return MIQ_OK;
    }
    const int64_t slices = max_slices(x.k);
    hipLaunchKernelGGL(column_max_kernel, dim3((unsigned) ((x.count + 255) / 256), (unsigned) slices), dim3(kBlock), 0, s,
                       x.p, x.ld, x.k, x.count, (x.k + slices - 1) / slices, largest, lost);
    MIQ_CHECK_LAUNCH();
    const int64_t tiles = ((x.count + 63) / 64) * ((kp + 63) / 64);
    MIQ_CHECK_ARG(tiles * kBlock <= UINT32_MAX, "an operand has too many tiles");
    hipLaunchKernelGGL(pack_columns_kernel, dim3((unsigned) tiles), dim3(kBlock), 0, s, x.p, x.ld, x.k, x.count, kp,
                       largest, (int) slices, (uint16_t*) to, exponents, lost);
    MIQ_CHECK_LAUNCH();
    return MIQ_OK;
}

// The operand as a kernel of 16-byte chunks reads it: as it lies, or copied to `at`, which then moves on
template <typename T, typename E>
int as_read(const Matrix<T>& x, int64_t bytes, char** at, Operand<E>* o, hipStream_t s)
{
    *o = {(const E*) x.p, x.ld, x.count};
    if (x.whole())
        return MIQ_OK;
    T* const to = (T*) *at;
    *o          = {(const E*) to, padded<T>(x.inner()), x.count};
    *at += bytes;
    return copy_rows(x.p, x.outer(), x.inner(), o->ld, to, s);
}

template <typename T, int ACT>
int launch_join(const float* partial, int splits, const Epilogue<T>& e, hipStream_t s)
{
    if (splits == 1)
        return MIQ_OK;
    const int64_t groups = (e.n + 7) / 8 * e.m;
    hipLaunchKernelGGL((join_kernel<T, ACT>), dim3((unsigned) ((groups + kBlock - 1) / kBlock)), dim3(kBlock), 0, s,
                       partial, splits, e);
    MIQ_CHECK_LAUNCH();
    return MIQ_OK;
}

template <typename T, int ACT, bool AC, bool BC>
int launch_product(Product<T>& p, bool big, hipStream_t s)
{
    const int tile = big ? 256 : 128;
    p.tiles_m = (int) ((p.e.m + tile - 1) / tile), p.tiles_n = (int) ((p.e.n + tile - 1) / tile);
    const int64_t blocks = (int64_t) p.tiles_m * p.tiles_n * p.splits;
    const dim3 grid((unsigned) blocks), threads(big ? 512 : 256);
    MIQ_CHECK_ARG(blocks * threads.x <= UINT32_MAX, "the product has too many tiles");
    if constexpr (std::is_same<T, float>::value)
    {
        if (big)
            hipLaunchKernelGGL((halves_kernel<ACT, 2, 4, 8, 4>), grid, threads, 0, s, p);
        else
            hipLaunchKernelGGL((halves_kernel<ACT, 2, 2, 4, 4>), grid, threads, 0, s, p);
    }
    else
    {
        if (big)
            hipLaunchKernelGGL((product_kernel<ACT, 2, 4, 8, 4, AC, BC>), grid, threads, 0, s, p);
        else
            hipLaunchKernelGGL((product_kernel<ACT, 2, 2, 4, 4, AC, BC>), grid, threads, 0, s, p);
    }
    MIQ_CHECK_LAUNCH();
    return launch_join<T, ACT>(p.partial, p.splits, p.e, s);
}

template <int ACT, bool AC, bool BC>
int launch_direct(DirectProduct& p, bool big, hipStream_t s)
{
    p.tiles_m = (int) ((p.e.m + (big ? 127 : 63)) / (big ? 128 : 64)), p.tiles_n = (int) ((p.e.n + 127) / 128);
    const int64_t blocks = (int64_t) p.tiles_m * p.tiles_n * p.splits;
    MIQ_CHECK_ARG(blocks * 256 <= UINT32_MAX, "the product has too many tiles");
    if (big)
        hipLaunchKernelGGL((direct_kernel<ACT, 2, 2, 4, 4, AC, BC>), dim3((unsigned) blocks), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((direct_kernel<ACT, 1, 4, 4, 2, AC, BC>), dim3((unsigned) blocks), dim3(256), 0, s, p);
    MIQ_CHECK_LAUNCH();
    return launch_join<float, ACT>(p.partial, p.splits, p.e, s);
}

template <typename T, int ACT>
int launch_few_rows(const T* a, const T* b, int64_t k, const Epilogue<T>& e, hipStream_t s)
{
    // about 2048 waves, each with 8 steps of k or more
    const int64_t blocks = (e.n + 15) / 16;
    int waves            = 4;
    while (waves < 16 && blocks * waves < 2048 && k / (4 * Chunk<T>::VEC) / (2 * waves) >= 8)
        waves *= 2;
    hipLaunchKernelGGL((few_rows_kernel<T, ACT>), dim3((unsigned) blocks), dim3(waves * 64), waves * 1024, s, a, b, k, e);
    MIQ_CHECK_LAUNCH();
    return MIQ_OK;
}

template <typename T>
int launch_few_rows_columns(const Matrix<T>& a, const Matrix<T>& b, const Plan& plan, float* partial,
                            const Epilogue<T>& e, hipStream_t s)
{
    constexpr int VEC  = IOTraits<T>::VEC, kWaves = 8;
    const int64_t wide = (b.count + 16 * VEC - 1) / (16 * VEC), per = (a.k + plan.splits - 1) / plan.splits;
    hipLaunchKernelGGL((few_rows_columns_kernel<T>), dim3((unsigned) wide, (unsigned) plan.splits), dim3(kWaves * 64),
                       kWaves * VEC * 1024, s, a.p, a.ld, b.p, a.k, per, plan.splits > 1 ? partial : nullptr, e);
    MIQ_CHECK_LAUNCH();
    return launch_join<T, MIQ_ACT_NONE>(partial, plan.splits, e, s);
}

// c[m, n] = act(sum over k of a(m, k) b(n, k) + bias) + residual
template <typename T, int ACT>
int product(const Matrix<T>& a, const Matrix<T>& b, const T* bias, const T* residual, T* c, Saved<T>* saved,
            char* workspace, hipStream_t s)
{
    if (a.count == 0 || b.count == 0)
        return MIQ_OK;
    constexpr bool kF32    = std::is_same<T, float>::value;
    const Plan plan        = plan_product(a, b);
    const Epilogue<T> e    = {bias, residual, c, saved, a.count, b.count};
    [[maybe_unused]] constexpr bool kPlain = ACT == MIQ_ACT_NONE;   // products of the backward pass, and some of the forward's
    if (plan.way == Way::kFewRows)
        return launch_few_rows<T, ACT>(a.p, b.p, a.k, e, s);
    if constexpr (kPlain)
        if (plan.way == Way::kFewColumns)
            return launch_few_rows_columns<T>(a, b, plan, (float*) workspace, e, s);
    if constexpr (kPlain && kF32)
        if (plan.way == Way::kShortSum)
        {
            const int64_t tiles = ((e.m + 127) / 128) * ((e.n + 127) / 128);
            MIQ_CHECK_ARG(tiles * kBlock <= UINT32_MAX, "the product has too many tiles");
            hipLaunchKernelGGL(short_sum_kernel, dim3((unsigned) tiles), dim3(kBlock), 0, s, a.p, a.ld, b.p, (int) a.k, e);
            MIQ_CHECK_LAUNCH();
            return MIQ_OK;
        }
    if constexpr (kF32)
        if (plan.way == Way::kDirect)
        {
            DirectProduct p = {{}, {}, a.k, 0, 0, plan.splits, nullptr, e};
            char* at        = workspace;
            if (int rc = as_read(a, plan.a_bytes, &at, &p.a, s))
                return rc;
            if (int rc = as_read(b, plan.b_bytes, &at, &p.b, s))
                return rc;
            p.partial = (float*) at;
            if constexpr (kPlain)
            {
                if (a.columns)
                    return launch_direct<ACT, true, true>(p, plan.big, s);
                if (b.columns)
                    return launch_direct<ACT, false, true>(p, plan.big, s);
            }
            return launch_direct<ACT, false, false>(p, plan.big, s);
        }
    Product<T> p = {};
    p.e          = e;
    p.splits     = plan.splits;
    char* at     = workspace;
    if constexpr (kF32)
    {
        char* const pb = at + plan.a_bytes;
        char* const sa = pb + plan.b_bytes;
        char* const sb = sa + plan.scale_a;
        if (int rc = pack(a, plan.kp, at, sa, s))
            return rc;
        if (int rc = pack(b, plan.kp, pb, sb, s))
            return rc;
        p.a       = {(const uint16_t*) at, 2 * plan.kp, a.count};
        p.b       = {(const uint16_t*) pb, 2 * plan.kp, b.count};
        p.k       = plan.kp;
        p.scale_a = (const int*) sa, p.scale_b = (const int*) sb;
        p.plain_a = {a.p, a.ld, a.columns}, p.plain_b = {b.p, b.ld, b.columns};
        p.length  = a.k;
        p.partial = (float*) (sb + plan.scale_b);
        return launch_product<T, ACT, false, false>(p, plan.big, s);
    }
    else
    {
        if (int rc = as_read(a, plan.a_bytes, &at, &p.a, s))
            return rc;
        if (int rc = as_read(b, plan.b_bytes, &at, &p.b, s))
            return rc;
        p.k       = a.k;
        p.partial = (float*) at;
        if constexpr (kPlain)
        {
            if (a.columns)
                return launch_product<T, ACT, true, true>(p, plan.big, s);
            if (b.columns)
                return launch_product<T, ACT, false, true>(p, plan.big, s);
        }
        return launch_product<T, ACT, false, false>(p, plan.big, s);
    }
}

template <typename T>
int64_t product_bytes(const Matrix<T>& a, const Matrix<T>& b)
{
    return a.count == 0 || b.count == 0 ? 0 : plan_product(a, b).total;
}

// The operands of the three products.  at16: x, w and grad start on multiples of 16 bytes.
template <typename T>
struct Operands
{
    int64_t rows, in, out;
    int activation;
    bool at16;

    Matrix<T> x_rows(const T* x) const
    {
        return {x, rows, in, false, at16, in};
    }
    Matrix<T> w_rows(const T* w) const
    {
        return {w, out, in, false, at16, in};
    }
    Matrix<T> x_columns(const T* x) const
    {
        return {x, in, rows, true, at16, in};
    }
    Matrix<T> w_columns(const T* w) const
    {
        return {w, in, out, true, at16, in};
    }
    // dz is grad itself, or is written to the workspace, in rows of whole chunks: where there is an activation, and where
    // grad would have to be copied anyway
    bool own_dz() const
    {
        return activation != MIQ_ACT_NONE || !at16 || padded<T>(out) != out;
    }
    int64_t dz_bytes() const
    {
        return own_dz() ? up256(rows * padded<T>(out) * (int64_t) sizeof(T)) : 0;
    }
    int64_t sums_bytes() const
    {
        return up256(slope_slices(rows, out) * out * (int64_t) sizeof(float));
    }
    Matrix<T> dz_rows(const T* dz) const
    {
        return {dz, rows, out, false, true, padded<T>(out)};
    }
    Matrix<T> dz_columns(const T* dz) const
    {
        return {dz, out, rows, true, true, padded<T>(out)};
    }
    int64_t forward_bytes() const
    {
        return product_bytes(x_rows(nullptr), w_rows(nullptr));
    }
    int64_t backward_bytes() const
    {
        return dz_bytes() + sums_bytes() + std::max(product_bytes(dz_rows(nullptr), w_columns(nullptr)),
                                                    product_bytes(dz_columns(nullptr), x_columns(nullptr)));
    }
};

template <typename T>
int linear_fwd(const T* x, const T* w, const T* bias, const T* residual, int64_t rows, int64_t in, int64_t out,
               int activation, T* y, void* saved, void* workspace, int64_t bytes, void* stream)
{
    if (int rc = check_shape(rows, in, out, activation))
        return rc;
    if (rows == 0 || out == 0)
        return MIQ_OK;
    MIQ_CHECK_ARG(y && (in == 0 || (x && w)), "null pointer");
    const Operands<T> o = {rows, in, out, activation, aligned(x) && aligned(w)};
    const int64_t need  = o.forward_bytes();
    MIQ_CHECK_ARG(bytes >= need && (workspace || need == 0), "the workspace is too small");
    MIQ_CHECK_ARG(need == 0 || (uintptr_t) workspace % 256 == 0, "the workspace is not aligned to 256 bytes");
    int rc = MIQ_OK;
    with_activation(activation, [&](auto act) {
        rc = product<T, act.value>(o.x_rows(x), o.w_rows(w), bias, residual, y, (Saved<T>*) saved,
                                   (char*) workspace, (hipStream_t) stream);
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
    const Operands<T> o = {rows, in, out, activation, aligned(g) && aligned(x) && aligned(w)};
    const int64_t need  = o.backward_bytes();
    MIQ_CHECK_ARG(bytes >= need && (workspace || need == 0), "the workspace is too small");
    MIQ_CHECK_ARG(need == 0 || (uintptr_t) workspace % 256 == 0, "the workspace is not aligned to 256 bytes");
    hipStream_t s  = (hipStream_t) stream;
    char* at       = (char*) workspace;
    T* own_dz      = o.own_dz() ? (T*) at : nullptr;
    const T* dz    = own_dz ? own_dz : g;
    float* partial = (float*) (at + o.dz_bytes());
    at += o.dz_bytes() + o.sums_bytes();
    const int64_t slices = slope_slices(rows, out);
    if ((own_dz || db) && out > 0)
    {
        const dim3 grid((unsigned) ((out + 255) / 256), (unsigned) slices);
        with_activation(activation, [&](auto act) {
            hipLaunchKernelGGL((slope_kernel<T, act.value>), grid, dim3(kBlock), 0, s, g, (const Saved<T>*) saved, rows, out,
                               padded<T>(out), (rows + slices - 1) / slices, own_dz, db ? partial : nullptr);
        });
        MIQ_CHECK_LAUNCH();
        if (db)
            hipLaunchKernelGGL(join_columns_kernel<T>, dim3((unsigned) ((out + 63) / 64)), dim3(kBlock), 0, s, partial, slices, out, db);
        MIQ_CHECK_LAUNCH();
    }
    int rc = MIQ_OK;
    if (dx)
        rc = product<T, MIQ_ACT_NONE>(o.dz_rows(dz), o.w_columns(w), nullptr, nullptr, dx, nullptr, at, s);
    if (rc == MIQ_OK && dw)
        rc = product<T, MIQ_ACT_NONE>(o.dz_columns(dz), o.x_columns(x), nullptr, nullptr, dw, nullptr, at, s);
    return rc;
}
}   // namespace
}   // namespace miq

using namespace miq;

extern "C"
{
int64_t miq_linear_workspace_bytes(int64_t rows, int64_t in_features, int64_t out_features, int activation, int bf16,
                                   int backward, int aligned)
{
    if (rows < 0 || in_features < 0 || out_features < 0)
        return 0;
    if (bf16)
    {
        const Operands<uint16_t> o = {rows, in_features, out_features, activation, aligned != 0};
        return backward ? o.backward_bytes() : o.forward_bytes();
    }
    const Operands<float> o = {rows, in_features, out_features, activation, aligned != 0};
    return backward ? o.backward_bytes() : o.forward_bytes();
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
