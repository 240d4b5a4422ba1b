// float32 products from operands cut into two halves beforehand (see pack_rows_kernel): coarse coarse + coarse fine + fine
// coarse, each through the half-precision matrix unit.
//
// A slice is 32 values of k, coarse halves and then fine ones: 128 bytes of a row, so that a slice is loaded and its
// fragments are read as those of 64 values of a 16-bit operand are ("half" 0 and 1 of the slice).  Every fragment read
// from LDS is multiplied three times for two here, where LDS reads, not the matrix unit, bound the 16-bit product.
// [4096, 4096] x [4096, 4096]^T: 270 us (1530 TFLOP/s through the matrix unit, 510 of float32), and 50 to make the halves;
// as three passes of the 16-bit product 328.  The relative error of the result is 2.5e-7 to 8e-7 there, where float32 matrix
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

    // Corrections are finite for finite operands.  Where an infinity or a NaN made a sum anything else, the coarse halves
    // alone say what comes out: those sums are formed once more, corrections first, cleared where they are not finite, and
    // the rest added.  The others are stored as they are.
    uint32_t bad[FM * FN / 8] = {};
    bool finite               = true;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (!__builtin_isfinite(acc[i][j][u]))
                {
                    bad[(i * FN + j) / 8] |= 1u << ((i * FN + j) % 8 * 4 + u);
                    finite = false;
                }
    const auto store = [&](auto again) {
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
                if constexpr (!decltype(again)::value)
                    finish_or_keep<float, ACT>(p, split, r, q, z);
                else
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if ((bad[(i * FN + j) / 8] >> ((i * FN + j) % 8 * 4 + u) & 1) && q + u < p.e.n)
                        {
                            if (p.splits == 1)
                                finish1<float, ACT>(p.e, r, q + u, z[u]);
                            else
                                p.partial[((int64_t) split * p.e.m + r) * p.e.n + q + u] = z[u];
                        }
            }
        }
    };
    store(std::false_type());
    if (__syncthreads_or(!finite))
    {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
        for (int pass = 0; pass < 2; ++pass)
        {
            rewind();
            for (int s = 0; s < count; ++s)
            {
                arrived();
                la.load(p.a, m0, lds0, wave, lane, LA::kDeep);
                lb.load(p.b, n0, lds0 + LA::kBytes, wave, lane, LB::kDeep);
                arrived();
                Columns c;
                read_columns(c, lds);
#pragma unroll
                for (int i = 0; i < FM; ++i)
                {
                    Row r;
                    read_row(r, lds, i);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        if (pass == 0)
                        {
                            acc[i][j] = mfma_16x16x32(c.coarse[j], r.fine, acc[i][j], half);
                            acc[i][j] = mfma_16x16x32(c.fine[j], r.coarse, acc[i][j], half);
                        }
                        else
                            acc[i][j] = mfma_16x16x32(c.coarse[j], r.coarse, acc[i][j], half);
                }
            }
            if (pass == 0)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            acc[i][j][u] = __builtin_isfinite(acc[i][j][u]) ? acc[i][j][u] : 0.f;
        }
        store(std::true_type());
    }
}
}   // namespace miq

#endif
