// Layer norm for gfx950: forward, and the backward pass with the reductions of the weight's and the bias' gradient.
//
//   m = mean(x), v = mean((x - m)^2), r = 1 / sqrt(v + eps), xhat = (x - m) r, y = xhat w + b
//   gw = g w, dx = r (gw - mean(gw) - xhat mean(gw xhat)), dw = sum over rows of g xhat, db = sum over rows of g
//
// All arithmetic is float32; only what is stored in bfloat16 is rounded to it, once.
//
// Nothing but reading and writing the rows counts: 2 passes over them forward, 3 backward, at the 5.1 TB/s that a large
// copy reaches.  16384 x 4096 bfloat16: forward 59 us (4.6 TB/s), backward 80 us and 7 to join the sums (4.6 TB/s);
// 8192 x 8192: forward 60 us; 8192 x 4096 float32: 50 us (5.3 TB/s).  Rows stay in registers, so each is read once.
#include "miq_io.h"

#include <algorithm>
#include <type_traits>

namespace miq
{
namespace
{
// sum over LANES threads (a wave, or a whole block of LANES), the same in each of them
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v, float* lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += __shfl_xor(v, o, 64);
    if constexpr (LANES > 64)
    {
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
            lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < LANES / 64; ++i)
            v += lds[i];
    }
    return v;
}

// Two sums at once.  The caller sees to it that everybody has read what `lds` held before.
template <int LANES>
__device__ __forceinline__ void lanes_sum2(float& a, float& b, float2* lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
    {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if constexpr (LANES > 64)
    {
        if ((threadIdx.x & 63) == 0)
            lds[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < LANES / 64; ++i)
        {
            a += lds[i].x;
            b += lds[i].y;
        }
    }
}

// A row lies in the registers of LANES threads, PER pieces of 16 bytes in each: piece i of lane l starts at value
// (i LANES + l) VEC.  The piece that reaches past the end starts earlier instead, so that it is whole, too: its first
// `twice` values are also those of the piece before, and are left out where the row is summed up (what is stored for them
// is stored twice, and the same).  Pieces altogether past the end are empty.  Only rows shorter than a piece are read value
// by value.
template <int VEC>
struct Piece
{
    int at, twice;
    bool has;

    __device__ __forceinline__ Piece(int c, int width)
    {
        has   = c < width;
        at    = c + VEC <= width || width < VEC ? c : width - VEC;
        twice = c - at;
    }
};

template <typename T>
__device__ __forceinline__ void load_piece(const T* p, int width, float* v)
{
    constexpr int VEC = IOTraits<T>::VEC;
    if (width >= VEC)
        load_any(p, v);
    else
#pragma unroll
        for (int u = 0; u < VEC; ++u)
            v[u] = u < width ? IOTraits<T>::load1(p + u) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, int width, const float* v)
{
    constexpr int VEC = IOTraits<T>::VEC;
    if (width >= VEC)
        store_any(p, v);
    else
#pragma unroll
        for (int u = 0; u < VEC; ++u)
            if (u < width)
                IOTraits<T>::store1(p + u, v[u]);
}

// the same as it lies in memory, and its values
template <typename T>
__device__ __forceinline__ any_u4 raw_piece(const T* p, int width)
{
    constexpr int VEC = IOTraits<T>::VEC;
    if (width >= VEC)
        return *(const any_u4*) p;
    T t[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u)
        t[u] = u < width ? p[u] : (T) 0;
    any_u4 v;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if constexpr (VEC == 4)
            v[u] = __float_as_uint(t[u]);
        else
            v[u] = (uint32_t) t[2 * u] | (uint32_t) t[2 * u + 1] << 16;
    return v;
}
__device__ __forceinline__ void values_of(any_u4 v, float (&f)[4])
{
#pragma unroll
    for (int u = 0; u < 4; ++u)
        f[u] = __uint_as_float(v[u]);
}
__device__ __forceinline__ void values_of(any_u4 v, float (&f)[8])
{
    IOTraits<uint16_t>::unpack(make_uint4(v[0], v[1], v[2], v[3]), f);
}
// One pass: the row stays in registers between its mean, its variance (from differences to the mean) and the result.
template <typename T, int PER, int LANES>
__global__ __launch_bounds__(LANES < kBlock ? kBlock : LANES) void ln_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, int64_t rows, int width, float eps,
    T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd)
{
    constexpr int VEC = IOTraits<T>::VEC, kRows = LANES < kBlock ? kBlock / LANES : 1;
    __shared__ float lds[LANES / 64];
    const int lane    = threadIdx.x % LANES;
    const int64_t row = block_index() * kRows + threadIdx.x / LANES;
    if (row >= rows)
        return;   // a whole wave, or, with one row a block, the whole block
    const T* px      = x + row * width;
    const bool whole = width % VEC == 0;   // the same for all: no piece starts earlier
    float v[PER][VEC], s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const Piece<VEC> piece((i * LANES + lane) * VEC, width);
#pragma unroll
        for (int u = 0; u < VEC; ++u)
            v[i][u] = 0.f;
        if (piece.has)
            load_piece(px + piece.at, width, v[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const Piece<VEC> piece((i * LANES + lane) * VEC, width);
        if (whole)
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                s += v[i][u];
        else
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                s += u < piece.twice ? 0.f : v[i][u];
    }
    const float m = lanes_sum<LANES>(s, lds) / (float) width;
    float q       = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const Piece<VEC> piece((i * LANES + lane) * VEC, width);
        if (!piece.has)
            continue;
        if (whole)
#pragma unroll
            for (int u = 0; u < VEC; ++u)
            {
                v[i][u] -= m;
                q = fmaf(v[i][u], v[i][u], q);
            }
        else
#pragma unroll
            for (int u = 0; u < VEC; ++u)
            {
                v[i][u] -= m;
                q = u >= piece.twice && (width >= VEC || u < width) ? fmaf(v[i][u], v[i][u], q) : q;
            }
    }
    const float r = 1.0f / sqrtf(lanes_sum<LANES>(q, lds) / (float) width + eps);
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const Piece<VEC> piece((i * LANES + lane) * VEC, width);
        if (!piece.has)
            continue;
        float ww[VEC], bb[VEC];
        if (w)
            load_piece(w + piece.at, width, ww);
        if (b)
            load_piece(b + piece.at, width, bb);
#pragma unroll
        for (int u = 0; u < VEC; ++u)
        {
            float h = v[i][u] * r;
            if (w)
                h *= ww[u];
            v[i][u] = b ? h + bb[u] : h;
        }
        store_piece(y + row * width + piece.at, width, v[i]);
    }
    if (lane == 0 && mean)
    {
        mean[row] = m;
        rstd[row] = r;
    }
}

// Rows too long for registers: read three times, the second and third from the caches
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                           const T* __restrict__ b, int64_t rows, int64_t width,
                                                           float eps, T* __restrict__ y, float* __restrict__ mean,
                                                           float* __restrict__ rstd)
{
    using IO = IOTraits<T>;
    __shared__ float lds[1024 / 64];
    const int64_t row = block_index();
    if (row >= rows)
        return;
    const T* px       = x + row * width;
    float s           = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += 1024)
        s += IO::load1(px + c);
    const float m = lanes_sum<1024>(s, lds) / (float) width;
    float q       = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += 1024)
    {
        const float d = IO::load1(px + c) - m;
        q             = fmaf(d, d, q);
    }
    const float r = 1.0f / sqrtf(lanes_sum<1024>(q, lds) / (float) width + eps);
    for (int64_t c = threadIdx.x; c < width; c += 1024)
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

// One pass over x and grad: a block takes rows block, block + blocks, ...; a thread meets the same columns in every row
// and keeps their sums g xhat and g.  partial[block][0][c] and [1][c] receive them, for ln_join_kernel.
// The next row is on its way while this one is worked on: as it lies in memory, which in bfloat16 takes half the registers.
template <typename T, int PER, int LANES>
__global__ __launch_bounds__(LANES < kBlock ? kBlock : LANES) void ln_bwd_kernel(
    const T* __restrict__ x, const T* __restrict__ g, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, int64_t rows, int width, T* __restrict__ dx, float* __restrict__ partial)
{
    constexpr int VEC = IOTraits<T>::VEC, kRows = LANES < kBlock ? kBlock / LANES : 1;
    __shared__ float2 lds[2][LANES / 64];
    const int lane = threadIdx.x % LANES;
    int odd        = 0;   // rows use the two halves of `lds` in turn: one barrier a row
    float sw[PER][VEC] = {}, sb[PER][VEC] = {};
    constexpr bool kHold = LANES < 1024 && PER <= 4;   // the weight stays in registers, where they allow it
    any_u4 nx[PER], ng[PER], rw[PER];
    float nm = 0.f, nr = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const Piece<VEC> piece((i * LANES + lane) * VEC, width);
        rw[i] = any_u4{0u, 0u, 0u, 0u};
        if (kHold && w && piece.has)
            rw[i] = raw_piece(w + piece.at, width);
    }
    const int64_t apart = (int64_t) gridDim.x * kRows;
    int64_t row         = (int64_t) blockIdx.x * kRows + threadIdx.x / LANES;
    const auto ask      = [&](int64_t at) {
        nm = mean[at];
        nr = rstd[at];
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            const Piece<VEC> piece((i * LANES + lane) * VEC, width);
            nx[i] = ng[i] = any_u4{0u, 0u, 0u, 0u};
            if (piece.has)
            {
                nx[i] = raw_piece(x + at * width + piece.at, width);
                ng[i] = raw_piece(g + at * width + piece.at, width);
            }
        }
    };
    if (row < rows)
        ask(row);
    for (; row < rows; row += apart)
    {
        const float m = nm, r = nr;
        float h[PER][VEC], gv[PER][VEC], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            values_of(nx[i], h[i]);
            values_of(ng[i], gv[i]);
        }
        if (row + apart < rows)
            ask(row + apart);
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            const Piece<VEC> piece((i * LANES + lane) * VEC, width);
            if (!piece.has)
                continue;
            float ww[VEC];
            if (kHold)
                values_of(rw[i], ww);
            else if (w)
                load_piece(w + piece.at, width, ww);
#pragma unroll
            for (int u = 0; u < VEC; ++u)
            {
                h[i][u] = (h[i][u] - m) * r;   // (past the end of a short row g is 0, and so is every sum's term)
                sw[i][u] = fmaf(gv[i][u], h[i][u], sw[i][u]);
                sb[i][u] += gv[i][u];
                if (w)
                    gv[i][u] *= ww[u];
                const float once = u < piece.twice ? 0.f : gv[i][u];
                s1 += once;
                s2 = fmaf(once, h[i][u], s2);
            }
        }
        if (!dx)
            continue;
        lanes_sum2<LANES>(s1, s2, lds[odd]);
        odd ^= 1;
        s1 /= (float) width;
        s2 /= (float) width;
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            const Piece<VEC> piece((i * LANES + lane) * VEC, width);
            if (!piece.has)
                continue;
#pragma unroll
            for (int u = 0; u < VEC; ++u)
                gv[i][u] = r * (gv[i][u] - s1 - h[i][u] * s2);
            store_piece(dx + row * width + piece.at, width, gv[i]);
        }
    }
    if (!partial)
        return;
    if constexpr (kRows > 1)
    {
        // the block's waves saw the same columns: added wave by wave
        __shared__ float both[2][PER * LANES * VEC];
        for (int k = 0; k < kRows; ++k)
        {
            if ((int) threadIdx.x / LANES == k)
#pragma unroll
                for (int i = 0; i < PER; ++i)
                {
                    const Piece<VEC> piece((i * LANES + lane) * VEC, width);
#pragma unroll
                    for (int u = 0; u < VEC; ++u)
                        if (piece.has && u >= piece.twice)
                        {
                            const int c = piece.at + u;
                            both[0][c]  = k ? both[0][c] + sw[i][u] : sw[i][u];
                            both[1][c]  = k ? both[1][c] + sb[i][u] : sb[i][u];
                        }
                }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < width; c += kBlock)
        {
            partial[((int64_t) blockIdx.x * 2) * width + c]     = both[0][c];
            partial[((int64_t) blockIdx.x * 2 + 1) * width + c] = both[1][c];
        }
    }
    else
    {
#pragma unroll
        for (int i = 0; i < PER; ++i)
        {
            const Piece<VEC> piece((i * LANES + lane) * VEC, width);
            if (!piece.has)
                continue;
#pragma unroll
            for (int k = 0; k < VEC; k += 4)
            {
                store_any(partial + ((int64_t) blockIdx.x * 2) * width + piece.at + k, sw[i] + k);
                store_any(partial + ((int64_t) blockIdx.x * 2 + 1) * width + piece.at + k, sb[i] + k);
            }
        }
    }
}

// rows too long for registers
template <typename T>
__global__ __launch_bounds__(1024) void ln_dx_long_kernel(const T* __restrict__ x, const T* __restrict__ g,
                                                          const T* __restrict__ w, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, int64_t rows,
                                                          int64_t width, T* __restrict__ dx)
{
    using IO = IOTraits<T>;
    __shared__ float2 lds[1024 / 64];
    const int64_t row = block_index();
    if (row >= rows)
        return;
    const T* px       = x + row * width;
    const T* pg       = g + row * width;
    const float m = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += 1024)
    {
        const float gw = IO::load1(pg + c) * (w ? IO::load1(w + c) : 1.f);
        s1 += gw;
        s2 = fmaf(gw, (IO::load1(px + c) - m) * r, s2);
    }
    lanes_sum2<1024>(s1, s2, lds);
    s1 /= (float) width;
    s2 /= (float) width;
    for (int64_t c = threadIdx.x; c < width; c += 1024)
    {
        const float gw = IO::load1(pg + c) * (w ? IO::load1(w + c) : 1.f);
        const float h  = (IO::load1(px + c) - m) * r;
        IO::store1(dx + row * width + c, r * (gw - s1 - h * s2));
    }
}

// column sums of a slice of the rows, for rows too long for registers
template <typename T>
__global__ __launch_bounds__(kBlock) void ln_dparams_long_kernel(const T* __restrict__ x, const T* __restrict__ g,
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
        sw             = fmaf(gv, (IO::load1(x + row * width + c) - mean[row]) * rstd[row], sw);
        sb += gv;
    }
    partial[((int64_t) blockIdx.y * 2) * width + c]     = sw;
    partial[((int64_t) blockIdx.y * 2 + 1) * width + c] = sb;
}

// adds partial[0 .. slices) of 32 columns, 32 threads a column, in an order that the number of slices alone decides
template <typename T>
__global__ __launch_bounds__(1024) void ln_join_kernel(const float* __restrict__ partial, int64_t slices,
                                                       int64_t width, T* __restrict__ dw, T* __restrict__ db)
{
    __shared__ float lds[32][33];
    const int64_t first = ((int64_t) blockIdx.z * gridDim.x + blockIdx.x) * 32, c = first + threadIdx.x % 32;
    const int part  = threadIdx.x / 32;
    T* out          = blockIdx.y == 0 ? dw : db;
    if (!out)
        return;
    float s = 0.f;
    if (c < width)
        for (int64_t k = part; k < slices; k += 32)
            s += partial[(k * 2 + blockIdx.y) * width + c];
    lds[part][threadIdx.x % 32] = s;
    __syncthreads();
    // thread (part, lane) now adds column `part`: value `lane`
    float v = lds[threadIdx.x % 32][part];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor(v, o, 64);
    const int64_t to = first + part;
    if (threadIdx.x % 32 == 0 && to < width)
        IOTraits<T>::store1(out + to, v);
}

// How a row is held: 32 values a thread at most, 16 with 1024 threads (the backward pass keeps four registers a value).
// Rows of up to 2048 values take a wave each, up to 8192 a block of 256, up to 16384 a block of 1024.
enum class Rows
{
    kWave,
    kBlock,
    kWide,
    kLong
};

Rows rows_of(int64_t width)
{
    return width <= 2048 ? Rows::kWave : width <= 8192 ? Rows::kBlock : width <= 16384 ? Rows::kWide : Rows::kLong;
}

// Blocks of the backward pass.  512 fill the device (16384 x 4096 bfloat16: 175 us with 256, 91 with 512, 93 with 768,
// 104 with 1024, whose partial sums cost more than they hide; blocks of 1024 threads: half as many), and no more than give
// each wave or block two rows (2048 x 1024 float32: 21 us with one row, 17 with two, 18 with four, 24 with eight).
int64_t ln_slices(int64_t rows, int64_t width)
{
    if (rows_of(width) == Rows::kLong)
    {
        const int64_t columns = (width + kBlock - 1) / kBlock;
        return std::max<int64_t>(1, std::min<int64_t>((1024 + columns - 1) / columns, rows / 16));
    }
    const int64_t each = rows_of(width) == Rows::kWave ? 8 : 2, most = rows_of(width) == Rows::kWide ? 256 : 512;
    return std::max<int64_t>(1, std::min<int64_t>(most, (rows + each - 1) / each));
}

// f(PER, LANES) as integral constants, for a row held in registers
template <typename T, typename F>
void with_rows(int64_t width, F&& f)
{
    const auto with_lanes = [&](auto lanes, auto most) {
        // all of a thread's pieces, half or a quarter of them: the fewest that hold the row
        constexpr int P     = decltype(most)::value / IOTraits<T>::VEC;
        const int64_t piece = (int64_t) decltype(lanes)::value * IOTraits<T>::VEC, need = (width + piece - 1) / piece;
        if (need > P / 2)
            f(std::integral_constant<int, P>(), lanes);
        else if (need > P / 4)
            f(std::integral_constant<int, P / 2>(), lanes);
        else
            f(std::integral_constant<int, P / 4 ? P / 4 : 1>(), lanes);
    };
    if (rows_of(width) == Rows::kWave)
        with_lanes(std::integral_constant<int, 64>(), std::integral_constant<int, 32>());
    else if (rows_of(width) == Rows::kBlock)
        with_lanes(std::integral_constant<int, 256>(), std::integral_constant<int, 32>());
    else
        with_lanes(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>());
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
    hipStream_t s  = (hipStream_t) stream;
    if (rows_of(width) == Rows::kLong)
        hipLaunchKernelGGL(ln_fwd_long_kernel<T>, grid_of(rows, 1024), dim3(1024), 0, s, x, w, b, rows, width, eps, y, mean,
                           rstd);
    else
        with_rows<T>(width, [&](auto per, auto lanes) {
            constexpr int P = decltype(per)::value, L = decltype(lanes)::value;
            constexpr int kRows = L < kBlock ? kBlock / L : 1, kThreads = L < kBlock ? kBlock : L;
            hipLaunchKernelGGL((ln_fwd_kernel<T, P, L>), grid_of((rows + kRows - 1) / kRows, kThreads),
                               dim3(kThreads), 0, s, x, w, b, rows, (int) width, eps, y, mean, rstd);
        });
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
    hipStream_t s        = (hipStream_t) stream;
    const int64_t slices = ln_slices(rows, width);
    float* partial       = dw || db ? workspace : nullptr;
    if (!dx && !partial)
        return MIQ_OK;
    if (rows_of(width) == Rows::kLong)
    {
        if (dx && rows)
            hipLaunchKernelGGL(ln_dx_long_kernel<T>, grid_of(rows, 1024), dim3(1024), 0, s, x, g, w, mean, rstd, rows,
                               width, dx);
        MIQ_CHECK_LAUNCH();
        if (partial)
            hipLaunchKernelGGL(ln_dparams_long_kernel<T>, dim3((unsigned) ((width + kBlock - 1) / kBlock), (unsigned) slices),
                               dim3(kBlock), 0, s, x, g, mean, rstd, rows, width, (rows + slices - 1) / slices, partial);
        MIQ_CHECK_LAUNCH();
    }
    else if (rows || partial)
    {
        with_rows<T>(width, [&](auto per, auto lanes) {
            constexpr int P = decltype(per)::value, L = decltype(lanes)::value;
            constexpr int kThreads = L < kBlock ? kBlock : L;
            hipLaunchKernelGGL((ln_bwd_kernel<T, P, L>), dim3((unsigned) slices), dim3(kThreads), 0, s, x, g, w,
                               mean, rstd, rows, (int) width, dx, partial);
        });
        MIQ_CHECK_LAUNCH();
    }
    if (partial)
    {
        const dim3 over = grid_of((width + 31) / 32, 1024);   // (y: weight and bias)
        hipLaunchKernelGGL(ln_join_kernel<T>, dim3(over.x, 2, over.y), dim3(1024), 0, s, partial, slices, width, dw, db);
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
