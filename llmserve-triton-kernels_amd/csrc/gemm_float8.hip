// Matrix products of rows in 8-bit floating point:  X[M,K] * W[N,K]^T with a scale per row of X and 128 columns and one per 128 rows and
// 128 columns of W (float8.h), 32-bit sums on the matrix cores, which apply the scales themselves:
//
//   plain    C[M,N] (+ bias), bfloat16 or float
//   gated    W = [gate; up]: C[M,N/2] = unit(gate) * up in 32 bits, rounded once: to bfloat16, or to rows in 8 bits for the next product
//   groups   rows seg[g] .. seg[g + 1] of X meet the weight W[g] (rows sorted by expert); tile_start[g]: tiles of 128 rows before group g
//
// A workgroup owns a tile of BM rows of X by BN rows of W and walks K in blocks of 128 columns, which come into one of two places in LDS by loads
// that go there directly: whole lines of 128 bytes (in halves of them the same bytes are twice as many requests to the L2, 3 % slower), a piece of
// 16 bytes to its place XOR half the row, so that the rows of a matrix operand are read without bank conflicts.  A lane's 32 bytes of
// v_mfma_scale_f32_32x32x64_f8f6f4 are two of the half's four pieces of its row, for both operands (which of the columns those are does not matter as
// long as both agree).  While a half of a block is multiplied the other one's operands are read, in an order that is written down (left to itself the
// compiler puts reads in front of what waits for them).  Blocks' scales of a row come four to a register, from which the instruction picks a byte.
//
// 8192 x 8192 x 8192 takes 400 microseconds, 2750 TFLOP/s, on four waves, which read LDS for half as many bytes a product as eight (433; with 256
// accumulators a lane in a register file of their own); 8192 x 57344 x 8192 2730, 2820 TFLOP/s; 2048 x 12288 x 4096 86 in tiles of 256 x 192.  The matrix
// instructions alone would take 220; without the loads of X and W it is 308.  The clock is at 1.76 GHz of 2.4 then, with the matrix
// instructions at work in 77 % of the cycles (524,000 of 682,000 at 8192 cubed): what the card draws bounds it, and next to that the L2.
//
// Few tiles of a long K are shared out in parts of K, whose sums a second kernel adds up in their order: 200 x 4096 x 14336 58 -> 30 microseconds.
//
// Those instructions add 16 products at a time and drop what lies more than 13 bits below the largest of them (one product of 2^16 and one of
// 2^3 come out exact, 2^2 is lost; measured, undocumented; sums of such sixteens are 32-bit's): 1.5e-5 of a result, in the mean, which
// is a 130th of what rounding it to bfloat16 takes and less of 8 bits.  A result in 32 bits, and any that a caller asks for so (`exact`), has its
// products from v_mfma_f32_32x32x16_bf16 at half the rate instead: values times their scales are bfloat16 numbers, exactly.  (8192 x 57344 x 8192 to 8
// bits 6220 microseconds and not 2730.)
#include "float8.h"

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) int i32x8;

#define G8_BF16 0
#define G8_FLOAT 1
#define G8_GATED 2
#define G8_GATED_8 3
#define G8_SUMS 4  // a part's sums, in 32 bits, of the 8-bit products (G8_FLOAT's: of exact ones)

// Tiles along M that are walked together.  An XCD's 32 compute units then work on 4 x 8 tiles (8192 x 8192 x 8192, with loads of half lines: 478, 465,
// 488, 545, 541 and 570 microseconds with 2, 4, 5, 8, 16 and 32).  Tiles of 64 rows: twice as many (8192 x 8192 x 4096 in such 368 and 388).
#define G8_BAND 4

struct Gemm8Args {
    const uint8_t *X, *XS, *W, *WS;
    const bf16* bias;
    void* C;
    uint8_t* CS;                 // GATED_8: the scales of the result
    long ldx, ldc;               // bytes of X, elements of C
    int ldxs, ldcs, s_cols;      // bytes from one row's scales to the next's: of X, of C, of W
    int M, N, K;                 // K: padded to 128
    int inter, unit;             // gated: rows of gate; the unit
    float limit;
    int tiles_m, tiles, band, band_tiles;
    int bias_fours;              // the bias is of whole fours
    const int *seg, *tile_start; // groups, or null
    int groups;
    int parts, part_blocks;      // of K, each a multiple of 4 blocks; C: [parts][M][ldc] where there are several
    long w_stride, ws_stride;    // bytes from one group's weight (scales) to the next's
};

// Row of W behind row `r` of the tile's columns: gated products take blocks of 32 rows of gate and of up in turn.
template <bool GATED>
__device__ __forceinline__ int g8_weight_row(const Gemm8Args& a, int r) {
    if constexpr (GATED) return ((r / 32) & 1) * a.inter + (r / 64) * 32 + r % 32;
    return r;
}

// The group whose tiles hold tile t: as many groups as have tile_start[g + 1] <= t lie in front of it.
__device__ __forceinline__ int g8_group(const int* __restrict__ tile_start, int groups, int t) {
    int g = 0;
    for (int base = 0; base < groups; base += LLMS_WAVE) {
        const int i = base + (int)threadIdx.x % LLMS_WAVE;
        g += __popcll(__ballot(i < groups && tile_start[i + 1] <= t));
    }
    return g;
}

// An address that is the same for all lanes, known to the compiler as such.
__device__ __forceinline__ const uint8_t* g8_uniform(const uint8_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
#else
    return p;
#endif
}

template <int SEL>
__device__ __forceinline__ f32x16 g8_mfma(const i32x8& w, const i32x8& x, const f32x16& c, int sw, int sx) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 0, 0, SEL, sw, SEL, sx);
#else
    return c;
#endif
}

template <int BM, int BN, int WM, int WN, int EPI, bool GROUPED>
__global__ __launch_bounds__(WM * WN * LLMS_WAVE) void gemm_float8_kernel(const Gemm8Args a) {
    constexpr bool GATED = EPI == G8_GATED || EPI == G8_GATED_8;
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int LM = BM / 8 / NW, LN = BN / 8 / NW;        // loads of 8 rows, per wave
    constexpr int SM = BM / LLMS_WAVE, SN = BN / LLMS_WAVE;  // loads of 64 rows' scales, of the workgroup
    static_assert(LM * NW * 8 == BM && LN * NW * 8 == BN && TM * WM * 32 == BM && TN * WN * 32 == BN && SM * LLMS_WAVE == BM && SN * LLMS_WAVE == BN,
                  "tile does not divide");
    static_assert(!GATED || TN % 2 == 0, "gate and up lie in one wave");
    static_assert(EPI != G8_GATED_8 || BN == 2 * F8_BLOCK, "a tile's units are one block");
    constexpr int SP = (SM + SN + NW - 1) / NW;              // of which a wave does as many
    constexpr int XT = BM * 128, STEP = XT + BN * 128, SCALES = (BM + BN) * 4;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];  // two blocks, then two times four blocks' scales
    uint8_t* const scales = lds + 2 * STEP;

    const int full = gridDim.x / 8, rem = gridDim.x % 8, xcd = blockIdx.x % 8, share = xcd * full + min(xcd, rem) + blockIdx.x / 8;
    const int part = share / a.tiles, t = share - part * a.tiles;
    int above = 0, in_band = t, high = a.tiles_m;
    if (a.band < a.tiles_m) {
        const int b = t / a.band_tiles;
        above = b * a.band;
        in_band = t - b * a.band_tiles;
        high = min(a.band, a.tiles_m - above);
    }
    int m0 = (above + in_band % high) * BM;
    const int n0 = in_band / high * BN;  // in rows of W as the tile takes them
    int m_end = a.M;
    const uint8_t *W = a.W, *WS = a.WS;
    if constexpr (GROUPED) {
        const int tile = m0 / BM;
        if (tile >= a.tile_start[a.groups]) return;
        const int g = __builtin_amdgcn_readfirstlane(g8_group(a.tile_start, a.groups, tile));
        m0 = a.seg[g] + (tile - a.tile_start[g]) * BM;
        m_end = min(a.seg[g + 1], a.M);
        if (m0 < 0 || m0 >= m_end) return;  // (no segment of these rows)
        W += g * a.w_stride;
        WS += g * a.ws_stride;
    }
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / LLMS_WAVE), lane = tid % LLMS_WAVE;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int r32 = lane % 32, hi = lane / 32;
    const int first = part * a.part_blocks, blocks = min(a.part_blocks, a.K / 128 - first);

    // A load brings 8 rows of 128 bytes, whole lines: lane l row l / 8, to place l.  A row's piece p of 16 bytes lies at its place p ^ (row / 2) % 8: two
    // rows are as wide as the 64 banks, and of 16 rows whose same piece is read at once no two then meet in a bank.  (Rows that do not exist are read
    // as ones that do: nothing of them is stored.)  Blocks beyond the last are asked for of buffers without bytes: zeros, no memory is touched.
    const int lr = lane / 8;
    unsigned off[LM + LN];
    f8_for<LM + LN>([&](auto i_) {
        constexpr bool ROWS = decltype(i_)::n < LM;
        const int r = (ROWS ? wave * LM + i_.n : wave * LN + i_.n - LM) * 8 + lr;
        const unsigned at = ((lane % 8) ^ (r / 2 % 8)) * 16;
        if constexpr (ROWS) off[i_.n] = (unsigned)(min(r, m_end - 1 - m0) * (int)a.ldx) + at;
        else off[i_.n] = (unsigned)min(g8_weight_row<GATED>(a, n0 + r), a.N - 1) * (unsigned)a.K + at;
    });
    const uint8_t *const x_base = g8_uniform(a.X + (size_t)m0 * a.ldx + first * 128), *const w_base = g8_uniform(W + first * 128);
    // load i of a block's LM + LN
    auto fetch = [&](int block, auto place, auto which) {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int i = decltype(which)::n;
        const unsigned bytes = (unsigned)__builtin_amdgcn_readfirstlane(block < blocks ? -1 : 0);
        const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(i < LM ? x_base : w_base), 0, bytes, 0x00020000);
        uint8_t* at = lds + decltype(place)::n * STEP + (i < LM ? (wave * LM + i) * 1024 : XT + (wave * LN + i - LM) * 1024);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)at, 16, off[i], block * 128, 0, 0);
#endif
    };
    // Four blocks' scales of the tile's rows, SP loads of 64 rows a wave (rows that do not exist have those of one that does).
    const uint8_t* scale_from[SP];
#pragma unroll
    for (int p = 0; p < SP; ++p) {
        const int i = min(wave + p * NW, SM + SN - 1);  // (a load more where they do not divide: the same bytes to the same place)
        if (i < SM) {
            scale_from[p] = a.XS + (size_t)min(m0 + i * LLMS_WAVE + lane, m_end - 1) * a.ldxs + first;
        } else {
            const int r = min(g8_weight_row<GATED>(a, n0 + (i - SM) * LLMS_WAVE + lane), a.N - 1);
            scale_from[p] = WS + (size_t)(r / F8_BLOCK) * a.s_cols + first;
        }
    }
    auto fetch_scales = [&](uint8_t* to, int four) {
#if defined(__HIP_DEVICE_COMPILE__)
        const int at = min(four, (blocks - 1) / 4) * 4;
#pragma unroll
        for (int p = 0; p < SP; ++p)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(scale_from[p] + at),
                                             (__attribute__((address_space(3))) void*)(to + min(wave + p * NW, SM + SN - 1) * 256), 4, 0, 0);
#endif
    };

    // acc[i][j][4 q + r]: column 8 q + 4 hi + r of block i of the weights, row r32 of block j of X
    f32x16 acc[TN][TM];
    f8_for<TN>([&](auto i) { f8_for<TM>([&](auto j) { acc[i.n][j.n] = (f32x16)(0.f); }); });
    int ws[TN], xs[TM], next_ws[TN], next_xs[TM];
    // scale register r of TN + TM
    auto read_scale = [&](const uint8_t* from, auto r) {
        constexpr int R = decltype(r)::n;
        if constexpr (R < TN) next_ws[R] = *reinterpret_cast<const int*>(from + (BM + wn + R * 32 + r32) * 4);
        else next_xs[R - TN] = *reinterpret_cast<const int*>(from + (wm + (R - TN) * 32 + r32) * 4);
    };
    auto take_scales = [&]() {
        f8_for<TN>([&](auto i) { ws[i.n] = next_ws[i.n]; });
        f8_for<TM>([&](auto j) { xs[j.n] = next_xs[j.n]; });
    };
    // Fragments of the half that is multiplied and of the next one, in two pieces each.
    f8_u32x4 wf[2][TN][2], xf[2][TM][2];
    // Where a lane reads: X and W, piece 0 and 1, of either half of the block, moved from place to place.  (Kept as they are: with an address for each
    // fragment and place the registers do not suffice.)
    uint32_t from[2][2][2];
    f8_for<8>([&](auto k_) {
        constexpr int k = decltype(k_)::n, H = k & 1, Q = k / 2 & 1;
        const int row = (k / 4 ? wn : wm) + r32;
        from[k / 4][Q][H] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (k / 4 ? XT : 0) + row * 128 +
                            (((4 * H + 2 * Q + hi) ^ (r32 / 2 & 7)) * 16);
        asm volatile("" : "+v"(from[k / 4][Q][H]));
    });
    auto move = [&](auto half, int by) {
        f8_for<4>([&](auto k) {
            from[k.n / 2][k.n % 2][half.n] += by;
            asm volatile("" : "+v"(from[k.n / 2][k.n % 2][half.n]));
        });
    };
    auto piece = [&](uint32_t at, auto offset) {
        return *reinterpret_cast<const __attribute__((address_space(3))) f8_u32x4*>(at + decltype(offset)::n);
    };
    auto read_w = [&](auto half, auto r) {  // piece r of 2 TN
        constexpr int H = decltype(half)::n, R = decltype(r)::n;
        wf[H][R / 2][R & 1] = piece(from[1][R & 1][H], Number<R / 2 * 4096>());
    };
    auto read_x = [&](auto half, auto r) {  // piece r of 2 TM
        constexpr int H = decltype(half)::n, R = decltype(r)::n;
        xf[H][R / 2][R & 1] = piece(from[0][R & 1][H], Number<R / 2 * 4096>());
    };
    auto operand = [&](const f8_u32x4 (&v)[2]) {
        return (i32x8){(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3], (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
    };
    // The products of a half.  `beside(q)`: what is read and asked for behind product q of TN TM, in this order: left to itself the compiler asks
    // for everything at once, which the wave then stands in front of, and reads at the end, where it waits for what it has read.
    auto multiply = [&](auto parity, auto sel, auto&& beside) {
        constexpr int SEL = decltype(sel)::n, H = decltype(parity)::n;
        if constexpr (EPI == G8_FLOAT) {
            f8_bf16x8 wv[TN][4];
            f8_for<TN>([&](auto i) {
                const float s = f8_scale(((uint32_t)ws[i.n] >> (8 * SEL)) & 255u);
                f8_for<4>([&](auto k) {  // (8 of a lane's 32 values at a time)
                    const f8_u32x4& v = wf[H][i.n][k.n / 2];
                    wv[i.n][k.n] = f8_numbers(v[k.n % 2 * 2], v[k.n % 2 * 2 + 1], s);
                });
            });
            f8_for<TM>([&](auto j) {
                const float s = f8_scale(((uint32_t)xs[j.n] >> (8 * SEL)) & 255u);
                f8_bf16x8 xv[4];
                f8_for<4>([&](auto k) {
                    const f8_u32x4& v = xf[H][j.n][k.n / 2];
                    xv[k.n] = f8_numbers(v[k.n % 2 * 2], v[k.n % 2 * 2 + 1], s);
                });
                f8_for<TN>([&](auto i) {
                    f8_for<4>([&](auto k) { acc[i.n][j.n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv[i.n][k.n], xv[k.n], acc[i.n][j.n], 0, 0, 0); });
                    beside(Number<decltype(j)::n * TN + decltype(i)::n>());
                });
            });
        } else {
            f8_for<TN * TM>([&](auto q) {
                constexpr int I = decltype(q)::n % TN, J = decltype(q)::n / TN;
                acc[I][J] = g8_mfma<SEL>(operand(wf[H][I]), operand(xf[H][J]), acc[I][J], ws[I], xs[J]);
                __builtin_amdgcn_sched_barrier(0);
                beside(q);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    };
    // waits until at most `left` loads of this wave are on their way and all that it reads of LDS is there, then for all waves
    auto arrive = [&](auto left) {
        constexpr int n = decltype(left)::n;
        static_assert(n < 64, "the counter of loads on their way");
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((n & 15) | ((n >> 4) << 14) | 0x0070);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int MULS = TN * TM, LOADS = LM + LN, READS = 2 * (TN + TM);
    // piece r of the READS of a half
    auto read = [&](auto half, auto r) {
        constexpr int R = decltype(r)::n;
        if constexpr (R < 2) read_w(half, r);
        else if constexpr (R < 2 + 2 * TM) read_x(half, Number<R - 2>());
        else read_w(half, Number<R - 2 * TM>());
    };
    // Block b (T of four).  While its first half is multiplied, the second is read, and then all waves have read the block: its place takes the
    // block after next, asked for beside the second half's products, while the next block's first half is read, which has been on its way for as
    // long as a half takes at least.  The scales of blocks 4 f .. 4 f + 3 are asked for two blocks ahead, and read beside the half in front of the
    // first that they are for.
    auto one = [&](int block, auto t) {
        constexpr int T = decltype(t)::n;
        multiply(Number<0>(), t, [&](auto q) {
            f8_for<READS>([&](auto r) {
                if constexpr (decltype(r)::n * (MULS * 3 / 4) / READS == decltype(q)::n) read(Number<1>(), r);
            });
        });
        arrive(Number<0>());
        move(Number<1>(), T & 1 ? -STEP : STEP);
        move(Number<0>(), T & 1 ? -STEP : STEP);
        if constexpr (T == 1) fetch_scales(scales + ((block / 4 + 1) % 2) * SCALES, block / 4 + 1);
        multiply(Number<1>(), t, [&](auto q) {
            constexpr int Q = decltype(q)::n;
            f8_for<READS>([&](auto r) {
                if constexpr (decltype(r)::n * MULS / READS == Q) read(Number<0>(), r);
            });
            f8_for<LOADS>([&](auto l) {
                if constexpr (decltype(l)::n * MULS / LOADS == Q) fetch(block + 2, Number<T & 1>(), l);
            });
            if constexpr (T == 3)
                f8_for<TN + TM>([&](auto r) {
                    if constexpr (decltype(r)::n * MULS / (TN + TM) == Q) read_scale(scales + ((block / 4 + 1) % 2) * SCALES, r);
                });
        });
        if constexpr (T == 3) take_scales();
    };
    fetch_scales(scales, 0);
    f8_for<2>([&](auto b) { f8_for<LOADS>([&](auto l) { fetch(b.n, b, l); }); });
    arrive(Number<LOADS>());
    f8_for<TN + TM>([&](auto r) { read_scale(scales, r); });
    f8_for<READS>([&](auto r) { read(Number<0>(), r); });
    take_scales();
    int block = 0;
    for (; block + 4 <= blocks; block += 4) f8_for<4>([&](auto t) { one(block + t.n, t); });
    f8_for<3>([&](auto t) {
        if (block + t.n < blocks) one(block + t.n, t);
    });
    __builtin_amdgcn_s_waitcnt(0);  // (no load may find the workgroup gone, nor what the epilogue keeps in LDS)
    asm volatile("" ::: "memory");

    // ---- a lane holds columns 8 q + 4 hi .. + 3 (q = 0 .. 3) of block i for row j * 32 + r32
    // A wave's rows, 32 at a time, go through LDS (16 bytes behind each, against bank conflicts) and out in whole pieces of 128 bytes and more: of stores
    // of the 4 columns that a lane holds, 8 bytes in each of 32 rows, 2048 x 12288 x 4096 takes 118 microseconds and not 88.
    constexpr bool FLOATS = EPI == G8_FLOAT || EPI == G8_SUMS;
    constexpr int OUT = GATED ? TN * 16 : TN * 32, SIZE = FLOATS ? 4 : 2, ROW = OUT * SIZE + 16, PIECES = OUT * SIZE / 16;
    static_assert(EPI == G8_GATED_8 || (NW * 32 * ROW <= 2 * STEP && 32 * PIECES % LLMS_WAVE == 0), "a wave's rows in LDS");
    // `four(j, c)`: the lane's columns 8 c + 4 hi .. + 3 of OUT
    auto store = [&](int n_wave, int cols, auto&& four) {
        uint8_t* const stage = lds + wave * 32 * ROW;
        f8_for<TM>([&](auto j) {
            f8_for<OUT / 8>([&](auto c) {
                const f32x4 v = four(j, c);
                uint8_t* to = stage + r32 * ROW + (8 * c.n + 4 * hi) * SIZE;
                if constexpr (FLOATS) *reinterpret_cast<f32x4*>(to) = v;
                else *reinterpret_cast<f8_u32x2*>(to) = (f8_u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            });
            // (LDS serves a wave in order)
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = lane; i < 32 * PIECES; i += LLMS_WAVE) {
                const int row = i / PIECES, piece = i % PIECES, m = m0 + wm + j.n * 32 + row, n = n_wave + piece * (16 / SIZE);
                const f8_u32x4 v = *reinterpret_cast<const f8_u32x4*>(stage + row * ROW + piece * 16);
                if (m >= m_end) continue;
                uint8_t* to = (uint8_t*)a.C + (((size_t)part * a.M + m) * a.ldc + n) * SIZE;
                if (n + 16 / SIZE <= cols) {
                    if constexpr (FLOATS) *reinterpret_cast<f8_u32x4_at4*>(to) = v;
                    else *reinterpret_cast<f8_u32x4_at2*>(to) = v;
                } else {
#pragma unroll
                    for (int r = 0; r < 16 / SIZE; ++r) {
                        if (n + r >= cols) continue;
                        if constexpr (FLOATS) reinterpret_cast<uint32_t*>(to)[r] = v[r];
                        else reinterpret_cast<uint16_t*>(to)[r] = (uint16_t)(v[r / 2] >> (16 * (r % 2)));
                    }
                }
            }
            asm volatile("" ::: "memory");
        });
    };
    __syncthreads();  // (every wave is done with the last block)
    if constexpr (!GATED) {
        // (all of a lane's columns of the bias are asked for at once; columns that do not exist take the last one's)
        f8_u32x2 bias[TN][4];
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int n = n0 + wn + i * 32 + 8 * q + 4 * hi;
                    if (a.bias_fours) {
                        bias[i][q] = *reinterpret_cast<const f8_u32x2_at2*>(a.bias + min(n, a.N - 4));
                    } else {
                        const uint16_t* from = reinterpret_cast<const uint16_t*>(a.bias);
                        bias[i][q] = (f8_u32x2){(uint32_t)from[min(n, a.N - 1)] | (uint32_t)from[min(n + 1, a.N - 1)] << 16,
                                                (uint32_t)from[min(n + 2, a.N - 1)] | (uint32_t)from[min(n + 3, a.N - 1)] << 16};
                    }
                }
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t lo = bias[i][q][0], up = bias[i][q][1];
#pragma unroll
                    for (int j = 0; j < TM; ++j) {
                        acc[i][j][4 * q] += __uint_as_float(lo << 16);
                        acc[i][j][4 * q + 1] += __uint_as_float(lo & 0xffff0000u);
                        acc[i][j][4 * q + 2] += __uint_as_float(up << 16);
                        acc[i][j][4 * q + 3] += __uint_as_float(up & 0xffff0000u);
                    }
                }
        }
        store(n0 + wn, a.N, [&](auto j, auto c) {
            constexpr int C = decltype(c)::n;
            const auto& v = acc[C / 4][decltype(j)::n];
            return (f32x4){v[C % 4 * 4], v[C % 4 * 4 + 1], v[C % 4 * 4 + 2], v[C % 4 * 4 + 3]};
        });
    } else {
        const int units = a.inter;
        // (units in place of the gates' sums; a loop for each, as a choice per number makes so much code of them that fetching it takes longer: 8192 x
        // 57344 x 8192 3170 microseconds and not 2760)
        auto unit = [&](auto which) {
#pragma unroll
            for (int p = 0; p < TN / 2; ++p)
#pragma unroll
                for (int j = 0; j < TM; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[2 * p][j][r] = f8_unit(acc[2 * p][j][r], acc[2 * p + 1][j][r], which.n, a.limit);
        };
        if (a.unit == 0) unit(Number<0>());
        else if (a.unit == 1) unit(Number<1>());
        else unit(Number<3>());
        if constexpr (EPI == G8_GATED) {
            store((n0 + wn) / 2, units, [&](auto j, auto c) {
                constexpr int C = decltype(c)::n;
                const auto& v = acc[C / 4 * 2][decltype(j)::n];
                return (f32x4){v[C % 4 * 4], v[C % 4 * 4 + 1], v[C % 4 * 4 + 2], v[C % 4 * 4 + 3]};
            });
        } else {
            // the largest of a row's 128 units: of the lane's, of the two lanes that hold the row, of the waves side by side
            constexpr int ROW8 = F8_BLOCK + 16;                    // (against bank conflicts)
            static_assert(WN * BM * 4 + BM * ROW8 <= 2 * STEP, "a tile's units in LDS");
            uint32_t* most_of = reinterpret_cast<uint32_t*>(lds);  // [WN][BM], then the rows of units
            uint8_t* const stage = lds + WN * BM * 4;
            auto most_units = [&](auto ragged_) {
                constexpr bool ragged = ragged_.n;
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    uint32_t most = 0;
#pragma unroll
                    for (int p = 0; p < TN / 2; ++p)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            if (ragged && (n0 + wn) / 2 + p * 32 + 8 * (r / 4) + 4 * hi + r % 4 >= units) acc[2 * p][j][r] = 0.f;
                            most = max(most, f8_magnitude(acc[2 * p][j][r]));
                        }
                    most = max(most, (uint32_t)__shfl_xor((int)most, 32, LLMS_WAVE));
                    if (hi == 0) most_of[(wave / WM) * BM + wm + j * 32 + r32] = most;
                }
            };
            if (n0 / 2 + F8_BLOCK <= units) most_units(Number<0>());
            else most_units(Number<1>());
            __syncthreads();
            const int unit_block = n0 / 2 / F8_BLOCK, last = (units + F8_BLOCK - 1) / F8_BLOCK - 1;
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const int row = wm + j * 32 + r32, m = m0 + row;
                uint32_t most = 0;
#pragma unroll
                for (int k = 0; k < WN; ++k) most = max(most, most_of[k * BM + row]);
                const uint32_t byte = f8_scale_byte(most);
                const float inv = f8_inverse(byte);
#pragma unroll
                for (int p = 0; p < TN / 2; ++p)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<uint32_t*>(stage + row * ROW8 + wn / 2 + p * 32 + 8 * q + 4 * hi) =
                            f8_pack4(acc[2 * p][j][4 * q] * inv, acc[2 * p][j][4 * q + 1] * inv, acc[2 * p][j][4 * q + 2] * inv,
                                     acc[2 * p][j][4 * q + 3] * inv);
                if (m >= m_end) continue;
                if (wn == 0 && hi == 0) {
                    uint8_t* s = a.CS + (size_t)m * a.ldcs;
                    s[unit_block] = (uint8_t)byte;
                    if (unit_block == last)  // (ones behind the last block)
                        for (int b = last + 1; b < 4 * (last / 4 + 1); ++b) s[b] = 127;
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = tid; i < BM * 8; i += NW * LLMS_WAVE) {
                const int row = i / 8, m = m0 + row;
                if (m < m_end)
                    *reinterpret_cast<f8_u32x4*>((uint8_t*)a.C + (size_t)m * a.ldc + n0 / 2 + i % 8 * 16) =
                        *reinterpret_cast<const f8_u32x4*>(stage + row * ROW8 + i % 8 * 16);
            }
        }
    }
}

// The parts' sums [parts][M][ld], added up in their order: a thread four columns (GATED: units) of a row.  Rows behind the last group's are left.
template <int EPI>
__global__ __launch_bounds__(256) void gemm_float8_parts_kernel(const Gemm8Args a, const float* sums, long ld, int quads) {
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(at / quads), n = 4 * (int)(at - (long)m * quads), cols = EPI == G8_GATED ? a.inter : a.N;
    if (m >= a.M || (a.seg && m >= a.seg[a.groups])) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f}, u = v;
    for (int p = 0; p < a.parts; ++p) {
        const float* from = sums + ((size_t)p * a.M + m) * ld + n;  // (rows end on 4)
        v += *reinterpret_cast<const f32x4*>(from);
        if constexpr (EPI == G8_GATED) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < cols) u[r] += from[a.inter + r];
        }
    }
    const bool whole = n + 4 <= cols;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if constexpr (EPI == G8_GATED) v[r] = f8_unit(v[r], u[r], a.unit, a.limit);
        else if (a.bias && n + r < cols) v[r] += to_f32(a.bias[n + r]);
    }
    if constexpr (EPI == G8_FLOAT) {
        float* c = (float*)a.C + (size_t)m * a.ldc + n;
        if (whole) {
            *reinterpret_cast<f8_u32x4_at4*>(c) = __builtin_bit_cast(f8_u32x4, v);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < cols) c[r] = v[r];
        }
    } else {
        bf16* c = (bf16*)a.C + (size_t)m * a.ldc + n;
        if (whole) {
            *reinterpret_cast<f8_u32x2_at2*>(c) = (f8_u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < cols) c[r] = from_f32<bf16>(v[r]);
        }
    }
}

template <int BM, int BN, int WM, int WN, int EPI, bool GROUPED>
static int g8_go(Gemm8Args& a, int m_tiles, hipStream_t stream) {
    const int cols = EPI == G8_GATED_8 || EPI == G8_GATED ? 64 * ((a.inter + 31) / 32) : a.N, n_tiles = (cols + BN - 1) / BN;
    a.tiles_m = m_tiles;
    const long tiles = (long)m_tiles * n_tiles;
    LLMS_REQUIRE(tiles * a.parts < (1l << 31), "gemm_float8: too many tiles");
    a.tiles = (int)tiles;
    constexpr int band = BM < 128 ? 2 * G8_BAND : G8_BAND;
    a.band = m_tiles <= band ? m_tiles : band;
    a.band_tiles = a.band * n_tiles;
    const int bytes = (BM + BN) * (2 * 128 + 2 * 4);
    auto kernel = gemm_float8_kernel<BM, BN, WM, WN, EPI, GROUPED>;
    static bool set[64] = {};
    if (const int failed = f8_raise_lds(reinterpret_cast<const void*>(kernel), bytes, set)) return failed;
    kernel<<<a.tiles * a.parts, WM * WN * LLMS_WAVE, bytes, stream>>>(a);
    LLMS_LAUNCH_CHECK();
}

// Tiles (bm, bn): 0 64 x 64, 1 128 x 128, 2 128 x 256, 3 256 x 256, 4 256 x 192 (EPI G8_BF16 alone).  Groups take 1, with the 128 rows of
// tile_start (GATED_8: 2); GATED_8, a block of whose units is 256 rows of W, takes 2 and 3; products in 32 bits, and sums, take 0 and 1 (more of
// them do not fit beside the operands).
template <int EPI, bool GROUPED>
static int g8_tile(int tile, Gemm8Args& a, hipStream_t stream) {
    const int mt = (a.M + 127) / 128 + a.groups;
    if constexpr (EPI == G8_GATED_8) {
        if (tile == 2) return g8_go<128, 256, 2, 4, EPI, GROUPED>(a, mt, stream);
    } else {
        if (tile == 1) return g8_go<128, 128, 2, 2, EPI, GROUPED>(a, mt, stream);
    }
    if constexpr (!GROUPED) {
        if constexpr (EPI != G8_GATED_8)
            if (tile == 0) return g8_go<64, 64, 2, 1, EPI, GROUPED>(a, (a.M + 63) / 64, stream);
        if constexpr (EPI != G8_FLOAT && EPI != G8_SUMS)
            if (tile == 3) return g8_go<256, 256, 2, 2, EPI, GROUPED>(a, (a.M + 255) / 256, stream);
        if constexpr (EPI == G8_BF16)
            if (tile == 4) return g8_go<256, 192, 4, 2, EPI, GROUPED>(a, (a.M + 255) / 256, stream);
    }
    LLMS_REQUIRE(false, "gemm_float8: no such tile");
}

// The sums of one part: of exact products, or (no groups then) of 8-bit ones.
template <bool GROUPED>
static int g8_sums(int tile, Gemm8Args& a, bool exact, hipStream_t stream) {
    if constexpr (!GROUPED)
        if (!exact) return g8_tile<G8_SUMS, false>(tile, a, stream);
    return g8_tile<G8_FLOAT, GROUPED>(tile, a, stream);
}

// The sums of the parts, then what is made of them.
template <int EPI, bool GROUPED>
static int g8_parts(int tile, Gemm8Args& a, void* c, long ldc, bool exact, hipStream_t stream) {
    Gemm8Args b = a;
    b.bias = nullptr;
    const long ld = ((long)a.N + 3) / 4 * 4;
    b.ldc = ld;
    if (const int failed = g8_sums<GROUPED>(tile, b, exact || EPI == G8_FLOAT, stream)) return failed;
    const float* sums = (const float*)a.C;
    a.C = c, a.ldc = ldc;
    const int quads = ((EPI == G8_GATED ? a.inter : a.N) + 3) / 4;
    gemm_float8_parts_kernel<EPI><<<(unsigned)(((long)a.M * quads + 255) / 256), 256, 0, stream>>>(a, sums, ld, quads);
    LLMS_LAUNCH_CHECK();
}

// epilogue: G8_BF16 to G8_GATED_8, or G8_SUMS, which leaves the parts' sums (or the one part's).  `k`: padded to 128.  Gated: n = 2 inter.  Parts of
// part_blocks (a multiple of 4) blocks of K, whose sums go to `sums` [parts][m][n up to a multiple of 4] where there are several (no GATED_8 then, and
// groups have one part), with G8_SUMS and with `exact`: sums of exact products whatever is made of them.
extern "C" int llms_gemm_float8(int tile, int epilogue, void* c, long ldc, void* cs, int ldcs, const void* x, long ldx, const void* xs, int ldxs,
                                const void* w, const void* ws, int s_cols, const void* bias, int m, int n, int k, int unit, float limit,
                                const int* seg, const int* tile_start, int groups, long w_stride, long ws_stride, int part_blocks, int exact,
                                void* sums, void* stream) {
    LLMS_REQUIRE(m > 0 && n > 0 && k > 0 && k % 128 == 0 && ldx < (1 << 23) && k < (1 << 23) && (long)n * k < (1l << 32) - (1 << 23), "gemm_float8 sizes");
    LLMS_REQUIRE(epilogue != G8_SUMS || (sums && !bias), "gemm_float8: sums have a place and no bias");
    LLMS_REQUIRE(epilogue < G8_GATED || n % 2 == 0, "gemm_float8: gate and up have the same rows");
    LLMS_REQUIRE(part_blocks > 0 && (part_blocks >= k / 128 || (sums && part_blocks % 4 == 0)), "gemm_float8 parts");
    LLMS_REQUIRE(!sums || epilogue != G8_GATED_8, "gemm_float8: no sums of results in 8 bits");
    LLMS_REQUIRE(!sums || !seg || (exact && part_blocks >= k / 128), "gemm_float8: sums of groups are exact products', in one part");
    LLMS_REQUIRE(!exact || sums || epilogue == G8_FLOAT, "gemm_float8: exact products of results in fewer bits have a place for their sums");
    Gemm8Args a = {};
    a.X = (const uint8_t*)x, a.XS = (const uint8_t*)xs, a.W = (const uint8_t*)w, a.WS = (const uint8_t*)ws;
    a.bias = (const bf16*)bias, a.C = sums ? sums : c, a.CS = (uint8_t*)cs;
    a.ldx = ldx, a.ldc = ldc, a.ldxs = ldxs, a.ldcs = ldcs, a.s_cols = s_cols;
    a.M = m, a.N = n, a.K = k, a.inter = epilogue >= G8_GATED ? n / 2 : 0, a.unit = unit, a.limit = limit, a.bias_fours = n % 4 == 0;
    a.seg = seg, a.tile_start = tile_start, a.groups = seg ? groups : 0, a.w_stride = w_stride, a.ws_stride = ws_stride;
    a.parts = (k / 128 + part_blocks - 1) / part_blocks, a.part_blocks = part_blocks;
    hipStream_t st = (hipStream_t)stream;
    if (epilogue == G8_SUMS) {
        a.ldc = ((long)n + 3) / 4 * 4;
        return seg ? g8_sums<true>(tile, a, exact, st) : g8_sums<false>(tile, a, exact, st);
    }
    if (seg && sums) {
        if (epilogue == G8_BF16) return g8_parts<G8_BF16, true>(tile, a, c, ldc, exact, st);
        if (epilogue == G8_GATED) return g8_parts<G8_GATED, true>(tile, a, c, ldc, exact, st);
        LLMS_REQUIRE(false, "gemm_float8: groups' results in 32 bits are their sums");
    }
    if (seg) {
        if (epilogue == G8_BF16) return g8_tile<G8_BF16, true>(tile, a, st);
        if (epilogue == G8_FLOAT) return g8_tile<G8_FLOAT, true>(tile, a, st);
        if (epilogue == G8_GATED) return g8_tile<G8_GATED, true>(tile, a, st);
        return g8_tile<G8_GATED_8, true>(tile, a, st);
    }
    if (sums) {
        if (epilogue == G8_BF16) return g8_parts<G8_BF16, false>(tile, a, c, ldc, exact, st);
        if (epilogue == G8_FLOAT) return g8_parts<G8_FLOAT, false>(tile, a, c, ldc, exact, st);
        return g8_parts<G8_GATED, false>(tile, a, c, ldc, exact, st);
    }
    if (epilogue == G8_BF16) return g8_tile<G8_BF16, false>(tile, a, st);
    if (epilogue == G8_FLOAT) return g8_tile<G8_FLOAT, false>(tile, a, st);
    if (epilogue == G8_GATED) return g8_tile<G8_GATED, false>(tile, a, st);
    return g8_tile<G8_GATED_8, false>(tile, a, st);
}
