// float32 products from operands cut into two halves beforehand (see pack_rows_kernel): coarse coarse + coarse fine + fine
// coarse, each through the half-precision matrix unit.
//
// A slice is 32 values of k, coarse halves and then fine ones: 128 bytes of a row, so that a slice is loaded and its
// fragments are read as those of 64 values of a 16-bit operand are ("half" 0 and 1 of the slice).  Every fragment read
// from LDS is multiplied three times for two here, where LDS reads, not the matrix unit, bound the 16-bit product.
// [4096, 4096] x [4096, 4096]^T: 305 us (1350 TFLOP/s through the matrix unit, 450 of float32), and 53 to make the halves.
// Three passes of the 16-bit product take a fifth longer.  The relative error of the result is 2.5e-7 to 8e-7 there, where float32 matrix
// instructions have 7e-7 to 1.3e-6.
#ifndef MIQ_HALVES_H
#define MIQ_HALVES_H

#include "miq_product.h"

namespace miq
{
constexpr int kHalves = 32;   // values of k in a slice

// where the coarse half of value k of a row lies; the fine one kHalves further
__device__ __forceinline__ int64_t place_of_half(int64_t k)
{
    return k / kHalves * (2 * kHalves) + k % kHalves;
}

constexpr int kZeroRow = -(1 << 30);   // what a row of zeros is said to have lost; more than a row has values

// Sums of a strip that are formed one by one; more take the matrix unit and 100 us.  The weight's gradient of
// [4096, 4096] x [4096, 4096]^T with a few such sums in one column of x: 409 us, 820 by strips alone, 397 without any.
constexpr int kFewSums = 16;

// 4 values of row r from k on, zeros from `to` on
__device__ __forceinline__ void load_plain(const Plain& x, int64_t r, int64_t k, int64_t to, float* v)
{
    if (!x.columns && k + 4 <= to)
        load_any(x.p + r * x.ld + k, v);
    else
#pragma unroll
        for (int t = 0; t < 4; ++t)
            v[t] = k + t < to ? x.p[x.columns ? (k + t) * x.ld + r : r * x.ld + k + t] : 0.f;
}

// Sums over k in [from, to) of 16 rows of a (lane l: row r, of l % 16) and 16 FN rows of b from q0 on (those past the end are the
// last one again: what they make is not stored), straight from memory, as float32.  Four values of k of a row a lane, as
// the first and second factor of four v_mfma_f32_16x16x4: which value of k meets which step is the same for both.
// It runs for few strips or for none: of [4096, 4096] x [4096, 4096]^T all of them take 2.6 ms, and 4.0 for the weight's gradient.
template <int FN>
__device__ __forceinline__ void float32_strip(const Plain a, int64_t r, const Plain b, int64_t q0, int64_t n, int64_t from,
                                                        int64_t to, int lane, f4* sums)
{
    constexpr int kUnroll = 4;
    int64_t rb[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j)
    {
        const int64_t q = q0 + row_of_b(j, lane % 16);
        rb[j]           = q < n ? q : n - 1;
        sums[j]         = f4{0.f, 0.f, 0.f, 0.f};
    }
    for (int64_t k0 = from; k0 < to; k0 += 16 * kUnroll)
    {
        float va[kUnroll][4], vb[kUnroll][FN][4];
#pragma unroll
        for (int s = 0; s < kUnroll; ++s)
        {
            const int64_t k = k0 + 16 * s + lane / 16 * 4;
            load_plain(a, r, k, to, va[s]);
#pragma unroll
            for (int j = 0; j < FN; ++j)
                load_plain(b, rb[j], k, to, vb[s][j]);
        }
#pragma unroll
        for (int s = 0; s < kUnroll; ++s)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    sums[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vb[s][j][t], va[s][t], sums[j], 0, 0, 0);
    }
}

// The sum of one row of a and one of b, the same in all lanes
__device__ __forceinline__ float float32_sum(const Plain a, int64_t r, const Plain b, int64_t q, int64_t from, int64_t to, int lane)
{
    const float* pa       = a.p + (a.columns ? r : r * a.ld);
    const float* pb       = b.p + (b.columns ? q : q * b.ld);
    const int64_t step_a = a.columns ? a.ld : 1, step_b = b.columns ? b.ld : 1;
    float s              = 0.f;
#pragma unroll 8
    for (int64_t k = from + lane; k < to; k += 64)
        s = fmaf(pa[k * step_a], pb[k * step_b], s);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        s += __shfl_xor(s, o, 64);
    return s;
}

template <int ACT, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM* WN * 64) void halves_kernel(const Product<float> p)
{
    constexpr int kWaves = WM * WN, kTM = WM * FM * 16, kTN = WN * FN * 16;
    using LA             = Loader<uint16_t, kTM, kWaves, false, 0>;
    using LB             = Loader<uint16_t, kTN, kWaves, false, 1>;
    constexpr auto half  = std::false_type();   // the matrix unit's type
    __shared__ __attribute__((aligned(1024))) char lds[2 * (LA::kBytes + LB::kBytes)];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int blocks = p.tiles_m * p.tiles_n, split = blockIdx.x / blocks;
    int tm, tn;
    tile_of_block(blockIdx.x % blocks, blocks, p.tiles_m, p.tiles_n, &tm, &tn);
    const int64_t m0 = (int64_t) tm * kTM, n0 = (int64_t) tn * kTN;
    const int slices = (int) (p.k / kHalves);
    const int first = (int) ((int64_t) slices * split / p.splits), last = (int) ((int64_t) slices * (split + 1) / p.splits);
    const int count = last - first;

    LA la;
    LB lb;
    Reader<false, 0, LA::kChunks> ra;
    Reader<false, 1, LB::kChunks> rb;
    ra.place(wm * FM * 16, lane);
    rb.place(wn * FN * 16, lane);
    const uint32_t lds0 = lds_address(lds);
    const auto buffer   = [&](int s) { return lds + (s & 1) * (LA::kBytes + LB::kBytes); };
    const auto place    = [&](int s) { return lds0 + (uint32_t) (s & 1) * (LA::kBytes + LB::kBytes); };
    const auto rewind   = [&] {
        la.start(p.a, m0, wave, lane);
        lb.start(p.b, n0, wave, lane);
        la.p += (int64_t) first * la.step;
        lb.p += (int64_t) first * lb.step;
    };

    // what the lane's rows lost, and the most that one of its columns did: read here, where nobody waits for it
    int lost_a[FM], lost_b = kZeroRow;
#pragma unroll
    for (int i = 0; i < FM; ++i)
    {
        const int64_t r = m0 + wm * FM * 16 + i * 16 + lane % 16;
        lost_a[i]       = r < p.e.m ? p.scale_a[p.e.m + r] : kZeroRow;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u)
        {
            const int64_t q = n0 + wn * FN * 16 + row_of_b(j, lane / 16 * 4 + u);
            lost_b          = max(lost_b, q < p.e.n ? p.scale_b[p.e.n + q] : kZeroRow);
        }

    f4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

    struct Columns
    {
        s8v coarse[FN], fine[FN];
    };
    struct Row
    {
        s8v coarse, fine;
    };
    const auto read_row = [&](Row& r, const char* from, int i) {
        r.coarse = ra.read(from, i, 0);
        r.fine   = ra.read(from, i, 1);
    };
    const auto read_columns = [&](Columns& c, const char* from) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
        {
            c.coarse[j] = rb.read(from + LA::kBytes, j, 0);
            c.fine[j]   = rb.read(from + LA::kBytes, j, 1);
        }
    };
    const auto multiply = [&](int i, const Row& r, const Columns& c) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = mfma_16x16x32(c.coarse[j], r.fine, acc[i][j], half);
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = mfma_16x16x32(c.fine[j], r.coarse, acc[i][j], half);
#pragma unroll
        for (int j = 0; j < FN; ++j)
            acc[i][j] = mfma_16x16x32(c.coarse[j], r.coarse, acc[i][j], half);
    };
    constexpr int kAll = LA::kLoads + LB::kLoads, kStarts = (kAll + FM - 2) / (FM - 1);
    const auto sum     = [&](auto inside) {
        // starts a few loads of the slice after s (the last slice once more, where there is none: nobody reads it)
        const auto start_some = [&](int i, int s) {
#pragma unroll
            for (int u = i * kStarts; u < (i + 1) * kStarts && u < kAll; ++u)
            {
                if (u < LA::kLoads)
                    la.template load_one<decltype(inside)::value>(u, p.a, m0, place(s + 1), wave, lane, LA::kDeep);
                else
                    lb.template load_one<decltype(inside)::value>(u - LA::kLoads, p.b, n0, place(s + 1) + LA::kBytes, wave,
                                                                  lane, LB::kDeep);
            }
        };
        Row row[2];
        // Rows 0 .. FM - 2 of a slice; the last one waits for the next slice, whose first fragments are read meanwhile
        const auto most = [&](const Columns& c, int s) {
            if (s + 1 < count)
            {
                la.p += la.step;
                lb.p += lb.step;
            }
#pragma unroll
            for (int i = 0; i + 1 < FM; ++i)
            {
                start_some(i, s);
                read_row(row[(i + 1) & 1], buffer(s), i + 1);
                multiply(i, row[i & 1], c);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const auto next = [&](const Columns& before, Columns& now, int s) {
            arrived();   // slice s has arrived, and everybody has read slice s - 1
            read_columns(now, buffer(s));
            read_row(row[0], buffer(s), 0);
            multiply(FM - 1, row[(FM - 1) & 1], before);
            __builtin_amdgcn_sched_barrier(0);
            most(now, s);
        };
        static_assert(FM % 2 == 0, "the last row and the next slice's first take different places");
        Columns c0, c1;
        rewind();
#pragma unroll
        for (int i = 0; i + 1 < FM; ++i)
            start_some(i, -1);
        arrived();
        read_columns(c0, buffer(0));
        read_row(row[0], buffer(0), 0);
        most(c0, 0);
        int s = 1;
        for (; s + 1 < count; s += 2)
        {
            next(c0, c1, s);
            next(c1, c0, s + 1);
        }
        if (s < count)
        {
            next(c0, c1, s);
            multiply(FM - 1, row[(FM - 1) & 1], c1);
        }
        else
            multiply(FM - 1, row[(FM - 1) & 1], c0);
        arrived();   // (the loads that nobody reads)
    };
    if (count > 0)
    {
        if (!la_edge(p, m0, n0, kTM, kTN))
            sum(std::true_type());
        else
            sum(std::false_type());
    }

    // Sums that are formed again, from float32 operands by float32 matrix instructions:
    // - what is not finite.  Corrections are finite for finite operands, but an infinity or a NaN makes them anything.
    // - what lost bits may have changed.  Scaled values are below 2^15, and one that lost bits is off by at most 2^-25: the
    //   sum by at most 2^-10 for each such value of its two rows.  That is allowed to be k / 4 times 2^-24 of the sum itself,
    //   and so of the sum of its terms' magnitudes, of which float32 arithmetic may lose k times 2^-24.  Of normally
    //   distributed rows of 4096 one in 15 has such a value, and one sum in 10^8 is then small enough to be formed again.
    // The others are stored as they are.
    static_assert(FN == 4 && FM <= 8, "16 bits a row of fragments, in two words");
    uint64_t again[2] = {};
    const float most  = 65536.0f / (float) p.length;
#pragma unroll
    for (int i = 0; i < FM; ++i)
    {
        const int64_t r  = m0 + wm * FM * 16 + i * 16 + lane % 16;
        const float weak = (float) (lost_a[i] + lost_b) * most;
        bool any         = false;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                any |= !(fabsf(acc[i][j][u]) >= weak) || !__builtin_isfinite(acc[i][j][u]);
        if (any && r < p.e.m)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                {
                    const int64_t q  = n0 + wn * FN * 16 + row_of_b(j, lane / 16 * 4 + u);
                    const float here = q < p.e.n ? (float) (lost_a[i] + p.scale_b[p.e.n + q]) * most : 0.f;
                    if (q < p.e.n && (!(fabsf(acc[i][j][u]) >= here) || !__builtin_isfinite(acc[i][j][u])))
                        again[i / 4] |= 1ull << (i % 4 * 16 + j * 4 + u);
                }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
    {
        const int64_t r = m0 + wm * FM * 16 + i * 16 + lane % 16;
        if (r >= p.e.m)
            continue;
        const int sr = p.scale_a[r];
#pragma unroll
        for (int j = 0; j < FN; j += 2)
        {
            const int64_t q = n0 + wn * FN * 16 + 16 * j + 8 * (lane / 16);
            if (q >= p.e.n)
                continue;
            float z[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                z[u] = ldexpf(acc[i][j + u / 4][u % 4], sr + (q + u < p.e.n ? p.scale_b[q + u] : 0));
            finish_or_keep<float, ACT>(p, split, r, q, z);
        }
    }
    const int64_t from = (int64_t) first * kHalves, to = (int64_t) last * kHalves < p.length ? (int64_t) last * kHalves : p.length;
    if (__builtin_amdgcn_ballot_w64((again[0] | again[1]) != 0) == 0)
        return;
    const auto put = [&](int64_t r, int64_t q, float z) {
        if (p.splits == 1)
            finish1<float, ACT>(p.e, r, q, z);
        else
            p.partial[((int64_t) split * p.e.m + r) * p.e.n + q] = z;
    };
    for (int i = 0; i < FM; ++i)
    {
        uint32_t marks = (uint32_t) ((i < 4 ? again[0] : again[1]) >> (i % 4 * 16)) & 0xffffu;   // 4 bits for each j
        if (__builtin_amdgcn_ballot_w64(marks != 0) == 0)
            continue;
        int count = __popc(marks);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            count += __shfl_xor(count, o, 64);
        const int64_t r0 = m0 + wm * FM * 16 + i * 16, q0 = n0 + wn * FN * 16, r = r0 + lane % 16;
        if (count <= kFewSums)
        {
            // the first lane's first mark, until there is none
            while (const uint64_t lanes = __builtin_amdgcn_ballot_w64(marks != 0))
            {
                const int l = __builtin_ctzll(lanes), bit = __builtin_ctz(__builtin_amdgcn_readlane(marks, l));
                const int64_t q = q0 + row_of_b(bit / 4, l / 16 * 4 + bit % 4);
                const float z   = float32_sum(p.plain_a, r0 + l % 16, p.plain_b, q, from, to, lane);
                if (lane == l)
                {
                    put(r, q, z);
                    marks &= marks - 1;
                }
            }
            continue;
        }
        f4 sums[FN];
        float32_strip<FN>(p.plain_a, r < p.e.m ? r : p.e.m - 1, p.plain_b, q0, p.e.n, from, to, lane, sums);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (marks >> (4 * j + u) & 1)
                    put(r, q0 + row_of_b(j, lane / 16 * 4 + u), sums[j][u]);
    }
}
}   // namespace miq

#endif
