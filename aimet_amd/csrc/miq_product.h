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
//
// What bounds it is LDS: of 256 x 256 tiles a wave's share is 128 x 64, and its fragments take three quarters of the LDS
// reads that the time of its matrix instructions allows, the loads' writes the rest (without loads the same loop runs at
// 1600 TFLOP/s, without LDS reads either at 1860).  Four waves of 128 x 128 read a third less and are 5 % slower: one wave
// a SIMD has nothing to cover its waits.  bfloat16, 4096 x 4096 from 4096: 101 us forward, 98 and 99 for the gradients
// (1360 to 1395 TFLOP/s); 8192 cubed 793, 758 and 740 us (1387, 1450 and 1485); [4096, 4096] x [11008, 4096]^T 276 us.
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

template <typename E>
struct Operand
{
    const E* p;
    int64_t ld;      // elements between rows ("rows") or between values of k ("columns"); a multiple of 8
    int64_t count;   // m or n
};

// Where the 16-byte chunk `c` of row `r` of a slice lies: exchanged within a row such that the lanes of one LDS access
// meet different banks.  `KEY` 0: A in rows (lanes read 8 consecutive rows), 1: B in rows (8 rows as row_of_b deals
// them), 2: A in columns (lanes read rows k .. k + 3 and k + 8 .. k + 11, at the same columns), 3: B in columns (the
// same, columns as row_of_b deals them).  float32: 4: rows (16 rows at a time), 5: columns (rows k, k + 8, k + 16, k + 24).
template <int KEY>
__device__ __forceinline__ int exchanged(int r, int c)
{
    if (KEY == 0)
        return c ^ (r & 7);
    if (KEY == 1)
        return c ^ ((r & 3) | ((r >> 1) & 4));
    if (KEY == 4)
        return c ^ (r >> 1 & 7);
    if (KEY == 5)
        return c ^ (r >> 3 & 3) * 4;
    return c ^ ((r & 3) * 4 + (r >> 3 & 1) * 2);
}
// rows this far apart exchange their chunks alike
template <int KEY>
constexpr int period()
{
    return KEY == 0 ? 8 : KEY == 5 ? 32 : 16;
}

// row of B's 16 FN row share that lane index i (0..15) of fragment j holds
__device__ __forceinline__ int row_of_b(int j, int i)
{
    return 32 * (j / 2) + 8 * (i / 4) + 4 * (j % 2) + i % 4;
}

// Loads from memory to LDS are written out as instructions: to the compiler the builtin is a store that any LDS read
// after it may depend on, and it puts a wait for the load before the read.  Nothing is returned in registers.  What makes
// the loads' results visible is arrived() alone: every wave waits for its own loads and reads, then for the other waves.
__device__ __forceinline__ uint32_t lds_address(const char* p)
{
    return (uint32_t) (uintptr_t) (__attribute__((address_space(3))) const char*) p;
}
__device__ __forceinline__ void arrived()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// One operand's slices: who loads what.  COUNT rows (m or n) of the tile, WAVES waves load, 1 KiB each at a time: load i
// of a wave is the (i WAVES + wave)th KiB of the slice.  A lane's place in its row of LDS is then the same in every load
// (but in float32 columns), and so is its offset from the load's first byte: one 32-bit register, everything else is the
// same for the whole wave.
template <typename E, int COUNT, int WAVES, bool COLUMNS, int KEY>
struct Loader
{
    static constexpr int kVec    = 16 / sizeof(E);
    static constexpr int kDeep   = 128 / sizeof(E);                           // values of k in a slice
    static constexpr int kChunks = COLUMNS ? COUNT / kVec : 8;                // 16-byte chunks of a row in LDS
    static constexpr int kRows   = COLUMNS ? kDeep : COUNT;                   // rows in LDS
    static constexpr int kAtOnce = 64 / kChunks;                              // rows of a load
    static constexpr int kLoads  = kRows / kAtOnce / WAVES;                   // loads of a wave
    static constexpr int kBytes  = COUNT * 128;
    static constexpr bool kAlike = WAVES * kAtOnce % period<KEY>() == 0;      // a lane's chunk is the same in every load
    static_assert(kRows % (kAtOnce * WAVES) == 0, "the slice is cut evenly");

    const E* p;          // first value of the slice, of the wave's first row in LDS; the same in all lanes
    int64_t step;        // to the next slice
    int64_t apart;       // between the rows of two loads
    uint32_t offset;     // of the lane's chunk, in bytes
    bool edge;           // the tile reaches past the operand's end

    __device__ __forceinline__ void start(const Operand<E>& o, int64_t first, int wave, int lane)
    {
        const int r = wave * kAtOnce, c = exchanged<KEY>(r + lane / kChunks, lane % kChunks);
        step   = COLUMNS ? o.ld * kDeep : kDeep;
        apart  = o.ld * (kAtOnce * WAVES);
        p      = o.p + r * o.ld + (COLUMNS ? first : first * o.ld);
        offset = (uint32_t) (lane / kChunks) * (uint32_t) (o.ld * sizeof(E)) + c * 16;
        edge   = first + COUNT > o.count;
    }

    // (m0 is listed as written, though the compiler says that it keeps no value there across statements: what it puts into m0
    // for an instruction of its own then stays behind the asm or before it)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    // Starts load i of a slice with `left` values of k remaining (from its first) into `lds` (an address in LDS).  INSIDE: all of the slice is
    // inside of the operand; otherwise what is not is read as zeros.
    template <bool INSIDE>
    __device__ __forceinline__ void load_one(int i, const Operand<E>& o, int64_t first, uint32_t lds, int wave, int lane,
                                             int64_t left)
    {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (i * WAVES + wave) * 1024);
        if (INSIDE)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to),
                         "v"(offset_of(i, wave, lane)), "s"(p + i * apart)
                         : "m0", "memory");
        else
        {
            const int r   = (i * WAVES + wave) * kAtOnce + lane / kChunks;
            const int c   = exchanged<KEY>(r, lane % kChunks) * kVec;
            const bool in = COLUMNS ? r < left && first + c < o.count : c < left && first + r < o.count;
            const char* from =
                in ? (const char*) (p + i * apart) + offset_of(i, wave, lane) : (const char*) &g_zero16;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from)
                         : "m0", "memory");
        }
    }
#pragma clang diagnostic pop

    __device__ __forceinline__ void load(const Operand<E>& o, int64_t first, uint32_t lds, int wave, int lane,
                                         int64_t left)
    {
        const bool inside = !edge && left >= kDeep;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            if (inside)
                load_one<true>(i, o, first, lds, wave, lane, left);
            else
                load_one<false>(i, o, first, lds, wave, lane, left);
        p += step;
    }

    __device__ __forceinline__ uint32_t offset_of(int i, int wave, int lane) const
    {
        if (kAlike)
            return offset;
        const int r = wave * kAtOnce + lane / kChunks, c = lane % kChunks;
        return offset + (exchanged<KEY>(r + i * WAVES * kAtOnce, c) - exchanged<KEY>(r, c)) * 16;
    }
};

// A wave's fragments of one operand, from row 0 of its share `first` of the tile's rows.  place() is the lane's part of
// the address, the same for all of them; the fragment's own part is a constant.
template <bool COLUMNS, int KEY, int CHUNKS>
struct Reader
{
    uint32_t at;

    __device__ __forceinline__ void place(int first, int lane)
    {
        if (!COLUMNS)
        {
            const int r = first + (KEY == 1 ? row_of_b(0, lane % 16) : lane % 16);
            at          = r * 128 + exchanged<KEY>(r, lane / 16) * 16;
        }
        else
        {
            // names 4 columns of row k
            const int k = lane / 16 * 8 + lane % 16 / 4, q = first + (KEY == 3 ? row_of_b(0, lane % 4 * 4) : lane % 4 * 4);
            at          = k * (CHUNKS * 16) + exchanged<KEY>(k, q / 8) * 16 + q % 8 * 2;
        }
    }

    // fragment i, k from 32 half
    __device__ __forceinline__ s8v read(const char* lds, int i, int half) const
    {
        if (!COLUMNS)   // rows i 16 further (B: where row_of_b has them), which leaves the exchange as it is
            return *(const s8v*) (lds + (at ^ half * 64) + (KEY == 1 ? row_of_b(i, 0) : i * 16) * 128);
        // columns further on are other chunks of the same row: bits that the lane's part does not have, exchanged alike
        const uint32_t from = (at ^ (KEY == 3 ? i / 2 * 64 : i * 32)) + (KEY == 3 ? i % 2 * 8 : 0) + half * (512 * CHUNKS);
        const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*) (lds + from));
        const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4v*) (lds + from + 64 * CHUNKS));
        // (as pairs of 32-bit registers, that the two reads fill the halves of one operand without a move)
        typedef int i2 __attribute__((ext_vector_type(2)));
        typedef int i4 __attribute__((ext_vector_type(4)));
        const i2 l = __builtin_bit_cast(i2, lo), h = __builtin_bit_cast(i2, hi);
        return __builtin_bit_cast(s8v, i4{l[0], l[1], h[0], h[1]});
    }
};

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

// One value of the result: bias, activation, residual, and z for the backward pass
template <typename T, int ACT>
__device__ __forceinline__ void finish1(const Epilogue<T>& e, int64_t r, int64_t q, float z)
{
    const int64_t at = r * e.n + q;
    if (e.bias)
        z += value_at(e.bias + q);
    if (e.saved)
        put_at(e.saved + at, z);
    z = act_value<ACT>(z);
    if (e.residual)
        z += value_at(e.residual + at);
    put_at(e.c + at, z);
}

// the same for 4 values of a float32 matrix
__device__ __forceinline__ void load4(const float* p, int64_t left, float* v)
{
    if (left >= 4)
        load_any(p, v);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = i < left ? p[i] : 0.f;
}
__device__ __forceinline__ void store4(float* p, int64_t left, const float* v)
{
    if (left >= 4)
        store_any(p, v);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left)
                p[i] = v[i];
}
template <int ACT>
__device__ __forceinline__ void finish4(const Epilogue<float>& e, int64_t r, int64_t q, float* z)
{
    const int64_t at = r * e.n + q, left = e.n - q;
    float t[4];
    if (e.bias)
    {
        load4(e.bias + q, left, t);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            z[i] += t[i];
    }
    if (e.saved)
        store4(e.saved + at, left, z);
    if (e.residual)
        load4(e.residual + at, left, t);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        z[i] = act_value<ACT>(z[i]) + (e.residual ? t[i] : 0.f);
    store4(e.c + at, left, z);
}

// A float32 operand as it lies
struct Plain
{
    const float* p;
    int64_t ld;
    bool columns;
};

template <typename T>
struct Product
{
    Operand<uint16_t> a, b;
    int64_t k;             // length of the sum (float32: padded to whole slices of kHalves)
    int tiles_m, tiles_n;
    int splits;            // the sum over k is cut into this many pieces, whose results go to `partial`
    float* partial;        // [splits][m][n]
    const int* scale_a;    // float32: exponents of the rows' scales and, behind them, what the rows lost (pack_rows_kernel)
    const int* scale_b;
    Plain plain_a, plain_b;   // float32: what the halves were made from
    int64_t length;           // float32: of the sum, not padded
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

// Whether a tile reaches past the end of a matrix
template <typename T>
__device__ __forceinline__ bool la_edge(const Product<T>& p, int64_t m0, int64_t n0, int tm, int tn)
{
    return m0 + tm > p.a.count || n0 + tn > p.b.count;
}

// 8 values of row r from column q on: finished, or kept as a piece of a sum
template <typename T, int ACT>
__device__ __forceinline__ void finish_or_keep(const Product<T>& p, int split, int64_t r, int64_t q, float* z)
{
    if (p.splits == 1)
        finish8<T, ACT>(p.e, r, q, z);
    else
        store8(p.partial + ((int64_t) split * p.e.m + r) * p.e.n + q, p.e.n - q, z);
}

// bfloat16
template <int ACT, int WM, int WN, int FM, int FN, bool AC, bool BC>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(const Product<uint16_t> p)
{
    using T              = uint16_t;
    constexpr int kWaves = WM * WN, kTM = WM * FM * 16, kTN = WN * FN * 16;
    constexpr int kKeyA = AC ? 2 : 0, kKeyB = BC ? 3 : 1;
    using LA             = Loader<uint16_t, kTM, kWaves, AC, kKeyA>;
    using LB             = Loader<uint16_t, kTN, kWaves, BC, kKeyB>;
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

    LA la;
    LB lb;
    la.start(p.a, m0, wave, lane);
    lb.start(p.b, n0, wave, lane);
    la.p += (int64_t) first * la.step;
    lb.p += (int64_t) first * lb.step;
    int64_t left       = p.k - (int64_t) first * kSlice;
    const auto advance = [&] {   // after a slice's loads: on to the next one
        la.p += la.step;
        lb.p += lb.step;
        left -= kSlice;
    };

    f4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

    Reader<AC, kKeyA, LA::kChunks> ra;
    Reader<BC, kKeyB, LB::kChunks> rb;
    ra.place(wm * FM * 16, lane);
    rb.place(wn * FN * 16, lane);
    struct Fragments
    {
        s8v a[FM], b[FN];
    };
    // What a wave does between two barriers, in steps of FN matrix instructions each: the rows of one half of a slice are
    // multiplied (fragments `f`), the other half's fragments (`next`) are read from LDS meanwhile, two or three a step and
    // none in the last quarter, so that they are there when the half ends; and the next slice's loads are started, spread
    // over the steps, for a wave that finds the load path full waits with its matrix instructions behind it.  The order
    // is fixed step by step: left to itself the compiler starts all loads first and waits for all reads at once.
    constexpr int kReads = (FM + FN + FM - FM / 4 - 1) / (FM - FM / 4), kAll = LA::kLoads + LB::kLoads,
                  kStarts = (kAll + FM - 1) / FM;
    const uint32_t lds0 = lds_address(lds);
    Fragments f0, f1;
    const auto half_slice = [&](auto multiplies, const Fragments& f, auto reads, Fragments& next, const char* from, int half,
                                auto starts, auto inside, uint32_t to) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
        {
            if constexpr (decltype(starts)::value)
#pragma unroll
                for (int u = i * kStarts; u < (i + 1) * kStarts && u < kAll; ++u)
                {
                    if (u < LA::kLoads)
                        la.template load_one<decltype(inside)::value>(u, p.a, m0, to, wave, lane, left);
                    else
                        lb.template load_one<decltype(inside)::value>(u - LA::kLoads, p.b, n0, to + LA::kBytes, wave, lane,
                                                                      left);
                }
            if constexpr (decltype(multiplies)::value)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = mfma_16x16x32(f.b[j], f.a[i], acc[i][j], std::true_type());
            if constexpr (decltype(reads)::value)
#pragma unroll
                for (int u = i * kReads; u < (i + 1) * kReads && u < FM + FN; ++u)
                {
                    if (u < FN)
                        next.b[u] = rb.read(from + LA::kBytes, u, half);
                    else
                        next.a[u - FN] = ra.read(from, u - FN, half);
                }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (decltype(starts)::value)
            advance();
    };
    const int count = last - first;
    const auto sum  = [&](auto inside) {
        constexpr auto yes = std::true_type();
        constexpr auto no  = std::false_type();
        const auto buffer  = [&](int s) { return lds + (s & 1) * (LA::kBytes + LB::kBytes); };
        const auto place   = [&](int s) { return lds0 + (uint32_t) (s & 1) * (LA::kBytes + LB::kBytes); };
        half_slice(no, f0, no, f0, nullptr, 0, yes, inside, place(0));
        arrived();
        if (count > 1)
            half_slice(no, f0, yes, f0, buffer(0), 0, yes, inside, place(1));
        else
            half_slice(no, f0, yes, f0, buffer(0), 0, no, inside, 0u);
        half_slice(yes, f0, yes, f1, buffer(0), 1, no, inside, 0u);
        for (int s = 1; s + 1 < count; ++s)
        {
            arrived();   // slice s has arrived, and everybody has read slice s - 1
            half_slice(yes, f1, yes, f0, buffer(s), 0, yes, inside, place(s + 1));
            half_slice(yes, f0, yes, f1, buffer(s), 1, no, inside, 0u);
        }
        if (count > 1)
        {
            arrived();
            half_slice(yes, f1, yes, f0, buffer(count - 1), 0, no, inside, 0u);
            half_slice(yes, f0, yes, f1, buffer(count - 1), 1, no, inside, 0u);
        }
        half_slice(yes, f1, no, f1, nullptr, 0, no, inside, 0u);
    };
    if (count > 0)
    {
        if (!la_edge(p, m0, n0, kTM, kTN) && p.k % kSlice == 0)
            sum(std::true_type());
        else
            sum(std::false_type());
    }

#pragma unroll
    for (int i = 0; i < FM; ++i)
    {
        const int64_t r = m0 + wm * FM * 16 + i * 16 + lane % 16;
        if (r >= p.e.m)
            continue;
#pragma unroll
        for (int j = 0; j < FN; j += 2)
        {
            const int64_t q = n0 + wn * FN * 16 + 16 * j + 8 * (lane / 16);
            if (q >= p.e.n)
                continue;
            float z[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                z[u] = acc[i][j + u / 4][u % 4];
            finish_or_keep<T, ACT>(p, split, r, q, z);
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
