// Tiled matrix product on the matrix cores of gfx950: C[m, n] = sum over k of A(m, k) B(n, k) with an epilogue.
//
// Operands are 16-bit (bfloat16, or the halves float32 is split into).  Each comes in one of two layouts: "rows", with
// k contiguous (A[m][k]), or "columns", with m or n contiguous (A[k][m]), so that a product and both products of its
// backward pass read the tensors as they lie.
//
// A block of WM x WN waves makes a tile of (WM FM 16) x (WN FN 16) values, 64 values of k at a time.  The slices go from
// memory to LDS without passing through registers (16 bytes a lane), into one of two buffers while the other is
// multiplied.  v_mfma_f32_16x16x32 takes, in lane l, 8 consecutive k (from 8 (l / 16)) of row l % 16 of each operand:
//   rows:    one 16-byte LDS read;
//   columns: two transposing 8-byte reads: within 16 lanes, lane 4 t + q names 4 columns of row t of a 4 x 16 block
//            and lane i receives column i.
// B's fragment is given as the first factor, so that a lane ends up with 4 consecutive n of one m: the epilogue reads and
// writes along rows of C.  Rows of B are dealt to fragments such that fragments j and j + 1 of a lane are 8 consecutive n
// (see row_of_b): 16-byte accesses on bfloat16, 64 contiguous bytes for each m.
#ifndef MIQ_PRODUCT_H
#define MIQ_PRODUCT_H

#include "miq_activation.h"
#include "miq_io.h"

#include <type_traits>

namespace miq
{
typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f4 mfma_16x16x32(s8v a, s8v b, f4 c, std::true_type /* bfloat16 */)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4 mfma_16x16x32(s8v a, s8v b, f4 c, std::false_type /* half */)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

constexpr int kSlice = 64;   // values of k in a slice: 128 bytes of a row

// 16 zero bytes: what lanes outside of an operand load
__device__ const uint4 g_zero16 = {0u, 0u, 0u, 0u};

struct Operand
{
    const uint16_t* p;
    int64_t ld;      // elements between rows ("rows") or between values of k ("columns"); a multiple of 8
    int64_t count;   // m or n
};

// Where the 16-byte chunk `c` of row `r` of a slice lies: exchanged within a row such that the lanes of one LDS access
// meet different banks.  `KEY` 0: A in rows (lanes read 8 consecutive rows), 1: B in rows (8 rows as row_of_b deals
// them), 2: columns (lanes read 4 or 8 rows, at the same columns).
template <int KEY>
__device__ __forceinline__ int exchanged(int r, int c)
{
    if (KEY == 0)
        return c ^ (r & 7);
    if (KEY == 1)
        return c ^ ((r & 3) | ((r >> 1) & 4));
    return c ^ ((r & 3) * 4);
}

// row of B's 16 FN row share that lane index i (0..15) of fragment j holds
__device__ __forceinline__ int row_of_b(int j, int i)
{
    return 32 * (j / 2) + 8 * (i / 4) + 4 * (j % 2) + i % 4;
}

// One operand's slices: who loads what, and the fragments.  COUNT rows (m or n) of the tile, WAVES waves load.
template <int COUNT, int WAVES, bool COLUMNS, int KEY>
struct Loader
{
    static constexpr int kChunks = (COLUMNS ? COUNT * 2 : kSlice * 2) / 16;   // 16-byte chunks of a row in LDS
    static constexpr int kRows   = COLUMNS ? kSlice : COUNT;
    static constexpr int kLoads  = kRows * kChunks / 64 / WAVES;              // 1 KiB loads of a wave
    static constexpr int kBytes  = COUNT * kSlice * 2;
    static_assert(kRows * kChunks % (64 * WAVES) == 0, "the slice is cut evenly");

    const uint16_t* p[kLoads];
    int k_of[kLoads];   // first k of the lane's chunk, within the slice
    bool in[kLoads];    // columns: the chunk is inside of the operand
    int64_t step;

    __device__ __forceinline__ void start(const Operand& o, int64_t first, int wave, int lane)
    {
        step = COLUMNS ? o.ld * kSlice : kSlice;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
        {
            const int at = (wave * kLoads + i) * 64 + lane, r = at / kChunks;
            const int c = exchanged<KEY>(r, at % kChunks);
            if (COLUMNS)
            {
                in[i]   = first + c * 8 < o.count;
                k_of[i] = r;
                p[i]    = in[i] ? o.p + r * o.ld + first + c * 8 : o.p;
            }
            else
            {
                // rows past the end read the last one: nothing made of them is stored
                const int64_t row = first + r < o.count ? first + r : o.count - 1;
                in[i]             = true;
                k_of[i]           = c * 8;
                p[i]              = o.p + row * o.ld + c * 8;
            }
        }
    }

    // Starts the loads of a slice with `left` values of k remaining (from its first) into `lds`
    template <bool TAIL>
    __device__ __forceinline__ void load(char* lds, int wave, int64_t left)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
        {
            const uint16_t* from = p[i];
            if ((TAIL && k_of[i] >= left) || (COLUMNS && !in[i]))
                from = (const uint16_t*) &g_zero16;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*) from,
                                             (__attribute__((address_space(3))) void*) (lds + (wave * kLoads + i) * 1024),
                                             16, 0, 0);
            p[i] += step;
        }
    }
};

// fragment of rows row(0..15) of a slice, k from 32 half
template <bool COLUMNS, int KEY, int CHUNKS>
__device__ __forceinline__ s8v fragment(const char* lds, int row_i, int row_q, int half, int lane)
{
    if (!COLUMNS)
    {
        // row_i: this lane's row of the tile
        const int c = exchanged<KEY>(row_i, half * 4 + lane / 16);
        return *(const s8v*) (lds + row_i * 128 + c * 16);
    }
    // row_q: first of the 4 columns that this lane names
    const int k = half * 32 + lane / 16 * 8 + (lane % 16) / 4;
    s8v out;
#pragma unroll
    for (int u = 0; u < 2; ++u)
    {
        const int kk = k + 4 * u;
        const int at = kk * (CHUNKS * 16) + exchanged<KEY>(kk, row_q / 8) * 16 + (row_q % 8) * 2;
        const s4v v  = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*) (lds + at));
        out[4 * u] = v[0], out[4 * u + 1] = v[1], out[4 * u + 2] = v[2], out[4 * u + 3] = v[3];
    }
    return out;
}

// What the backward pass keeps of z = x w^T + b.  float32 tensors keep it as it is.  bfloat16 ones keep a half: as
// many bytes, three bits more, and z matters only through act'(z), which is flat far out, so saturating at the
// largest half loses nothing.  A z > 0 too small for a half is kept as the smallest one: ReLU's derivative goes by
// its sign.  NaN stays NaN.
template <typename T>
using Saved = std::conditional_t<std::is_same<T, float>::value, float, _Float16>;

__device__ __forceinline__ float kept_z(float z, float*)
{
    return z;
}
__device__ __forceinline__ _Float16 kept_z(float z, _Float16*)
{
    const float c = z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z;
    return (_Float16) (z > 0.f && z < 0x1p-24f ? 0x1p-24f : c);
}

// 8 consecutive values between memory and float32, at any address; of the last of a row only `left`
typedef _Float16 any_h8 __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ float value_at(const float* p)
{
    return *p;
}
__device__ __forceinline__ float value_at(const uint16_t* p)
{
    return bf16_to_f32(*p);
}
__device__ __forceinline__ float value_at(const _Float16* p)
{
    return (float) *p;
}
__device__ __forceinline__ void put_at(float* p, float v)
{
    *p = v;
}
__device__ __forceinline__ void put_at(uint16_t* p, float v)
{
    *p = (uint16_t) f32_to_bf16(v);
}
__device__ __forceinline__ void put_at(_Float16* p, float v)
{
    *p = kept_z(v, (_Float16*) nullptr);
}
__device__ __forceinline__ void load_whole8(const float* p, float* v)
{
    load_any(p, v);
    load_any(p + 4, v + 4);
}
__device__ __forceinline__ void load_whole8(const uint16_t* p, float* v)
{
    load_any(p, v);
}
__device__ __forceinline__ void load_whole8(const _Float16* p, float* v)
{
    const any_h8 h = *(const any_h8*) p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = (float) h[i];
}
__device__ __forceinline__ void store_whole8(float* p, const float* v)
{
    store_any(p, v);
    store_any(p + 4, v + 4);
}
__device__ __forceinline__ void store_whole8(uint16_t* p, const float* v)
{
    store_any(p, v);
}
__device__ __forceinline__ void store_whole8(_Float16* p, const float* v)
{
    any_h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        h[i] = kept_z(v[i], (_Float16*) nullptr);
    *(any_h8*) p = h;
}

template <typename S>
__device__ __forceinline__ void load8(const S* p, int64_t left, float* v)
{
    if (left >= 8)
        load_whole8(p, v);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = i < left ? value_at(p + i) : 0.f;
}
template <typename S>
__device__ __forceinline__ void store8(S* p, int64_t left, const float* v)
{
    if (left >= 8)
        store_whole8(p, v);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left)
                put_at(p + i, v[i]);
}

// Where z goes: y = act(z + bias) + residual, z + bias itself for the backward pass
template <typename T>
struct Epilogue
{
    const T* bias;        // or null
    const T* residual;    // or null
    T* c;
    Saved<T>* saved;      // or null
    int64_t m, n;
};

// z: 8 values of row r < m from column q < n on
template <typename T, int ACT>
__device__ __forceinline__ void finish8(const Epilogue<T>& e, int64_t r, int64_t q, float* z)
{
    const int64_t at = r * e.n + q, left = e.n - q;
    float t[8];
    if (e.bias)
    {
        load8(e.bias + q, left, t);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            z[i] += t[i];
    }
    if (e.saved)
        store8(e.saved + at, left, z);
    if (e.residual)
        load8(e.residual + at, left, t);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        z[i] = act_value<ACT>(z[i]) + (e.residual ? t[i] : 0.f);
    store8(e.c + at, left, z);
}

template <typename T>
struct Product
{
    Operand a, b;
    int64_t k;             // length of the sum (float32: padded to whole slices)
    int tiles_m, tiles_n;
    int splits;            // the sum over k is cut into this many pieces, whose results go to `partial`
    float* partial;        // [splits][m][n]
    const int* scale_a;    // float32: exponents of the rows' scales (see split_rows_kernel)
    const int* scale_b;
    Epilogue<T> e;
};

// Tile of a block.  Blocks go round the 8 XCDs in turn; each XCD gets a contiguous run of tiles, and within the run
// tiles go down 4 rows of tiles before they move right, so that the 32 blocks an XCD holds at a time share about 4 + 8
// operand panels in its L2.
__device__ __forceinline__ void tile_of_block(int block, int blocks, int tiles_m, int tiles_n, int* tm, int* tn)
{
    const int per = blocks / 8, more = blocks % 8, x = block % 8;
    int t           = x * per + (x < more ? x : more) + block / 8;
    const int band  = 4 * tiles_n, g = t / band;
    const int height = tiles_m - g * 4 < 4 ? tiles_m - g * 4 : 4;
    t -= g * band;
    *tm = g * 4 + t % height;
    *tn = t / height;
}

template <typename T, int ACT, int WM, int WN, int FM, int FN, bool AC, bool BC>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(const Product<T> p)
{
    constexpr bool kF32  = std::is_same<T, float>::value;
    constexpr int kWaves = WM * WN, kTM = WM * FM * 16, kTN = WN * FN * 16;
    using LA             = Loader<kTM, kWaves, AC, AC ? 2 : 0>;
    using LB             = Loader<kTN, kWaves, BC, BC ? 2 : 1>;
    using Kind           = std::integral_constant<bool, !kF32>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * (LA::kBytes + LB::kBytes)];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int blocks = p.tiles_m * p.tiles_n;
    const int split  = blockIdx.x / blocks;
    int tm, tn;
    tile_of_block(blockIdx.x % blocks, blocks, p.tiles_m, p.tiles_n, &tm, &tn);
    const int64_t m0 = (int64_t) tm * kTM, n0 = (int64_t) tn * kTN;

    const int slices = (int) ((p.k + kSlice - 1) / kSlice);
    const int first = (int) ((int64_t) slices * split / p.splits), last = (int) ((int64_t) slices * (split + 1) / p.splits);
    // float32: three passes over k, A's coarse halves with B's fine ones, fine with coarse, coarse with coarse
    const int count = (last - first) * (kF32 ? 3 : 1);

    LA la;
    LB lb;
    la.start(p.a, m0, wave, lane);
    lb.start(p.b, n0, wave, lane);
#pragma unroll
    for (int i = 0; i < LA::kLoads; ++i)
        la.p[i] += (int64_t) first * la.step;
#pragma unroll
    for (int i = 0; i < LB::kLoads; ++i)
        lb.p[i] += (int64_t) first * lb.step + (kF32 ? p.k : 0);
    int64_t left = p.k - (int64_t) first * kSlice;
    int issued   = 0;
    const auto issue = [&](int buffer) {
        char* to = lds + buffer * (LA::kBytes + LB::kBytes);
        if (left >= kSlice)
        {
            la.template load<false>(to, wave, left);
            lb.template load<false>(to + LA::kBytes, wave, left);
        }
        else
        {
            la.template load<true>(to, wave, left);
            lb.template load<true>(to + LA::kBytes, wave, left);
        }
        left -= kSlice;
        ++issued;
        if (kF32 && (issued == last - first || issued == 2 * (last - first)))
        {
            const int64_t back = (int64_t) (last - first) * kSlice;
            left += back;
            const int64_t ja = (issued == last - first ? p.k : -p.k) - back;
            const int64_t jb = (issued == last - first ? -p.k : 0) - back;
#pragma unroll
            for (int i = 0; i < LA::kLoads; ++i)
                la.p[i] += ja;
#pragma unroll
            for (int i = 0; i < LB::kLoads; ++i)
                lb.p[i] += jb;
        }
    };

    f4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

    const int i16 = lane % 16;
    if (count > 0)
        issue(0);
    for (int s = 0; s < count; ++s)
    {
        __syncthreads();   // slice s has arrived, and everybody is done with slice s - 1
        if (s + 1 < count)
            issue((s + 1) & 1);
        const char* sa = lds + (s & 1) * (LA::kBytes + LB::kBytes);
        const char* sb = sa + LA::kBytes;
        // the two passes over fine halves are corrections, finite for finite operands: where an infinity or a NaN
        // made them anything else, the coarse pass alone says what comes out
        if (kF32 && s == 2 * (last - first))
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        acc[i][j][u] = __builtin_isfinite(acc[i][j][u]) ? acc[i][j][u] : 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
            s8v fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i)
                fa[i] = fragment<AC, AC ? 2 : 0, LA::kChunks>(sa, wm * FM * 16 + i * 16 + i16,
                                                             wm * FM * 16 + i * 16 + (lane % 4) * 4, half, lane);
#pragma unroll
            for (int j = 0; j < FN; ++j)
                fb[j] = fragment<BC, BC ? 2 : 1, LB::kChunks>(sb, wn * FN * 16 + row_of_b(j, i16),
                                                             wn * FN * 16 + row_of_b(j, (lane % 4) * 4), half, lane);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = mfma_16x16x32(fb[j], fa[i], acc[i][j], Kind());
        }
    }

#pragma unroll
    for (int i = 0; i < FM; ++i)
    {
        const int64_t r = m0 + wm * FM * 16 + i * 16 + i16;
        if (r >= p.e.m)
            continue;
        const int sr = kF32 ? p.scale_a[r] : 0;
#pragma unroll
        for (int j = 0; j < FN; j += 2)
        {
            const int64_t q = n0 + wn * FN * 16 + 16 * j + 8 * (lane / 16);
            if (q >= p.e.n)
                continue;
            float z[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
            {
                z[u] = acc[i][j + u / 4][u % 4];
                if (kF32)
                    z[u] = ldexpf(z[u], sr + (q + u < p.e.n ? p.scale_b[q + u] : 0));
            }
            if (p.splits == 1)
                finish8<T, ACT>(p.e, r, q, z);
            else
                store8(p.partial + ((int64_t) split * p.e.m + r) * p.e.n + q, p.e.n - q, z);
        }
    }
}

// adds the pieces of a split sum, in order, and finishes
template <typename T, int ACT>
__global__ __launch_bounds__(kBlock) void join_kernel(const float* __restrict__ partial, int splits,
                                                      const Epilogue<T> e)
{
    const int64_t groups = (e.n + 7) / 8, at = (int64_t) blockIdx.x * kBlock + threadIdx.x;
    if (at >= groups * e.m)
        return;
    const int64_t r = at / groups, q = at % groups * 8;
    float z[8] = {};
    for (int s = 0; s < splits; ++s)
    {
        float t[8];
        load8(partial + ((int64_t) s * e.m + r) * e.n + q, e.n - q, t);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            z[i] += t[i];
    }
    finish8<T, ACT>(e, r, q, z);
}
}   // namespace miq

#endif
