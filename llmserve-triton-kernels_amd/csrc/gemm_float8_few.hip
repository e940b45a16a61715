// Products of few rows in 8-bit floating point against weights in 8 bits (gemm_float8.hip says which): decoding.  What bounds them is reading the weight.
//
//   gemm_float8_stream   one weight and up to 64 rows: a workgroup a compute unit, with X in its registers; described where it begins
//   gemm_float8_join     the sums of its parts of K
//   gemm_float8_few      a weight per group of rows, of up to 8 in the mean; described here
//
// A workgroup of 8 waves owns TN blocks of 16 rows of a group's weight and walks the group's rows 16 at a time, reading the weight anew for each 16: groups
// far above the mean take as many passes as they have sixteens, which stand behind one another.  Its waves share K out in blocks of 128, wave w
// takes blocks w, w + 8, ..., and meet in LDS in the order of the waves.  Weights come straight from memory into the registers of the matrix
// instruction: a lane takes the pieces g and g + 4 of 16 bytes of its row's 128 (g = lane / 16), so an instruction reads 64 bytes of
// each of 16 rows in one piece, and X is read the same way.
//
// X in bfloat16 becomes 8 bits on the way in (in the stream too): a lane has 32 of the 128 numbers of its row, the block's largest is two exchanges between
// the four lanes of the row away, and the conversion divides by the scale itself (v_cvt_scalef32_pk_fp8_bf16).  Every workgroup does that
// for itself: some 90 vector instructions per block of 128 columns and 16 rows, where another launch in front costs more.
#include "float8.h"

typedef __attribute__((ext_vector_type(4))) float f32x4;

#define G8_BF16 0
#define G8_FLOAT 1
#define G8_GATED 2

#define F8_NW 8

struct Few8Args {
    const void* X;               // 8 bits, or bfloat16
    const uint8_t *XS, *W, *WS;
    const bf16* bias;
    void* C;
    long ldx, ldc;               // elements
    int ldxs, s_cols;
    int M, N, K, blocks;         // K: of X in bfloat16; blocks of 128
    int kp;                      // 128 blocks: bytes of a weight row
    int inter, unit;
    float limit;
    int out_float;
    const int* seg;              // groups, or null
    long w_stride, ws_stride;
};

// 32 values of a row's block, with the block's scale, as four operands of v_mfma_f32_16x16x32_bf16.  (Which of the 128 columns an operand
// holds does not matter as long as both sides agree.)
struct Numbers32 {
    f8_bf16x8 v[4];
};
__device__ __forceinline__ Numbers32 numbers32(const f8_u32x4& lo, const f8_u32x4& hi, uint32_t byte) {
    const float s = f8_scale(byte);
    return {{f8_numbers(lo[0], lo[1], s), f8_numbers(lo[2], lo[3], s), f8_numbers(hi[0], hi[1], s), f8_numbers(hi[2], hi[3], s)}};
}

// 32 bfloat16 numbers of a row's block, which four lanes (16 apart) hold together, to 8 bits: values in the order of `v`, the block's byte.
__device__ __forceinline__ void rounded32(const f8_u32x4 (&v)[4], f8_u32x4 (&q)[2], uint32_t& byte) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    typedef __attribute__((ext_vector_type(2))) short s16x2;
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t magnitudes = v[i][j] & 0x7fff7fffu;
            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, magnitudes));
        }
    uint32_t m = max((uint32_t)most[0], (uint32_t)most[1]) << 16;
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, LLMS_WAVE));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, LLMS_WAVE));
    byte = f8_scale_byte(m);
    const float s = f8_scale(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t a = v[i][2 * j], b = v[i][2 * j + 1];
            s16x2 r = {0, 0};
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, a), s, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), s, true);
            q[i / 2][2 * (i % 2) + j] = byte == 255u ? 0x7f7f7f7fu : __builtin_bit_cast(uint32_t, r);
        }
#endif
}

template <int TN, int TM, int EPI, bool XB>
__global__ __launch_bounds__(F8_NW * LLMS_WAVE) void gemm_float8_few_kernel(const Few8Args a) {
    constexpr bool GATED = EPI == G8_GATED;
    static_assert(!GATED || TN % 2 == 0, "gate and up lie in one workgroup");
    extern __shared__ __attribute__((aligned(16))) f32x4 sums[];  // [F8_NW][TN][TM][64]
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / LLMS_WAVE), lane = tid % LLMS_WAVE;
    const int r16 = lane % 16, g = lane / 16;
    const int m_begin = a.seg[blockIdx.y], m_end = min(a.seg[blockIdx.y + 1], a.M);
    if (m_begin < 0 || m_begin >= m_end) return;  // (none, or no segment of these rows)
    const uint8_t *W = a.W + blockIdx.y * a.w_stride, *WS = a.WS + blockIdx.y * a.ws_stride;
    const int n0 = blockIdx.x * TN * 16;  // (GATED: blocks of gate and of up in turn)
    const uint8_t *wp[TN], *wsp[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        int r = GATED ? (i & 1) * a.inter + (n0 / 32 + i / 2) * 16 + r16 : n0 + i * 16 + r16;
        r = min(r, a.N - 1);  // (rows that do not exist: nothing of them is stored)
        wp[i] = W + (size_t)r * a.kp + 16 * g;
        wsp[i] = WS + (size_t)(r / F8_BLOCK) * a.s_cols;
    }
    for (int m0 = m_begin; m0 < m_end; m0 += 16 * TM) {
        const void* xp[TM];
        const uint8_t* xsp[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int m = min(m0 + j * 16 + r16, m_end - 1);
            if constexpr (XB) {
                xp[j] = (const bf16*)a.X + (size_t)m * a.ldx;
            } else {
                xp[j] = (const uint8_t*)a.X + (size_t)m * a.ldx + 16 * g;
                xsp[j] = a.XS + (size_t)m * a.ldxs;
            }
        }
        f32x4 acc[TN][TM];
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int b = wave; b < a.blocks; b += F8_NW) {
            f8_u32x4 lo[TN], hi[TN];
            uint32_t sw[TN];
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const uint8_t* p = wp[i] + (size_t)b * 128;
                lo[i] = *reinterpret_cast<const f8_u32x4*>(p);
                hi[i] = *reinterpret_cast<const f8_u32x4*>(p + 64);
                sw[i] = wsp[i][b];
            }
            Numbers32 x[TM];
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                if constexpr (XB) {
                    f8_u32x4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // (pieces of 8 numbers: 2 g, 2 g + 1, 8 + 2 g, 9 + 2 g of the block's 16)
                        const int c = b * 128 + (i / 2) * 64 + 16 * g + (i % 2) * 8;
                        v[i] = (f8_u32x4){0, 0, 0, 0};
                        if (c < a.K) v[i] = *reinterpret_cast<const f8_u32x4*>((const bf16*)xp[j] + c);
                    }
                    f8_u32x4 q[2];
                    uint32_t byte;
                    rounded32(v, q, byte);
                    x[j] = numbers32(q[0], q[1], byte);
                } else {
                    const uint8_t* p = (const uint8_t*)xp[j] + (size_t)b * 128;
                    x[j] = numbers32(*reinterpret_cast<const f8_u32x4*>(p), *reinterpret_cast<const f8_u32x4*>(p + 64), xsp[j][b]);
                }
            }
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const Numbers32 w = numbers32(lo[i], hi[i], sw[i]);
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[s], x[j].v[s], acc[i][j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) sums[((wave * TN + i) * TM + j) * LLMS_WAVE + lane] = acc[i][j];
        __syncthreads();
        // a thread adds up a lane's 4 sums of a block (GATED: of a block of gate and the block of up of the same units)
        constexpr int ITEMS = (GATED ? TN / 2 : TN) * TM * LLMS_WAVE;
        for (int at = tid; at < ITEMS; at += F8_NW * LLMS_WAVE) {
            const int l = at % LLMS_WAVE, j = at / LLMS_WAVE % TM, i = at / LLMS_WAVE / TM;
            const int m = m0 + j * 16 + l % 16;
            f32x4 v = {0.f, 0.f, 0.f, 0.f}, u = v;
#pragma unroll
            for (int w = 0; w < F8_NW; ++w) {
                v += sums[((w * TN + (GATED ? 2 * i : i)) * TM + j) * LLMS_WAVE + l];
                if constexpr (GATED) u += sums[((w * TN + 2 * i + 1) * TM + j) * LLMS_WAVE + l];
            }
            if (m >= m_end) continue;
            const int n = (GATED ? n0 / 2 : n0) + i * 16 + 4 * (l / 16), cols = GATED ? a.inter : a.N;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (GATED) {
                    v[r] = f8_unit(v[r], u[r], a.unit, a.limit);
                } else {
                    if (a.bias && n + r < cols) v[r] += to_f32(a.bias[n + r]);
                }
            }
            if constexpr (EPI == G8_FLOAT) {
                float* c = (float*)a.C + (size_t)m * a.ldc + n;
                if (n + 4 <= cols) {
                    *reinterpret_cast<f8_u32x4_at4*>(c) = __builtin_bit_cast(f8_u32x4, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < cols) c[r] = v[r];
                }
            } else {
                bf16* c = (bf16*)a.C + (size_t)m * a.ldc + n;
                if (n + 4 <= cols) {
                    *reinterpret_cast<f8_u32x2_at2*>(c) = (f8_u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < cols) c[r] = from_f32<bf16>(v[r]);
                }
            }
        }
        __syncthreads();  // (the sums' places are free for the next rows)
    }
}

// ------------------------------------------------------------------------------ a workgroup a compute unit
// One weight, X in registers: a workgroup owns a share of the weight rows (gated: of the units), a wave every eighth block of 128 columns of K,
// XC of them, whose part of X it holds (in 8 bits: 8 registers a block and 16 rows; as numbers, in twice as many, where they suffice) for all
// of the share.  It walks the share in tiles of
// 16 rows (gated: 8 units, gate in rows 0 to 7 of the matrix instruction and up in 8 to 15).  A block of a tile is 2 KB that come by
// loads which go to LDS directly, 8 rows of 128 bytes an instruction (as operands a row's bytes would be asked for in two pieces of 64), into
// one of NI places of the wave's own: NI blocks a wave are always on their way, through the ends of tiles; eight waves ask for 1 KB of a row side by
// side.  A piece of 16 bytes lies at its place XOR half the row, so that the operands are read without bank conflicts.  The waves' sums meet in
// LDS, in the order of the waves, in two places that take turns: a barrier a tile.
// More of K than eight waves hold of X is shared out to `parts` workgroups, whose sums a second kernel adds up in their order.
//
// EIGHT: bfloat16 results of more than 16 rows are of the 8-bit products (gemm_float8.hip says what those drop), others of bfloat16 ones, which are exact:
// 64 x 4096 x 11008 20 and 22 microseconds.
//
// What bounds it: memory, 57344 x 8192 gated for one row in 80 microseconds, 5.9 TB/s; smaller weights some 4 microseconds of start and end,
// 4096 x 4096 in 6.7, 12288 x 4096 in 12.3, and with more rows each workgroup's reading of X, 12288 x 4096 in 20.8 for 64.  (With blocks of a wave beside
// each other, 128 bytes of a row asked for at a time every 512, 12288 x 4096 takes 13.4.)
struct Stream8Args {
    Few8Args a;
    int quads, each, more;   // units of the product in fours; a share has `each`, the first `more` one more
    int parts, part_blocks;  // of K; blocks of 128 of one
    float* sums;             // [parts][M][ld], gate and up (each up to a multiple of 4) side by side; null: one part
    int ld, up_at;
    unsigned x_bytes, xs_bytes;  // from the first byte of X (its scales) to behind the last
};

// what is made of a lane's four sums (n .. n + 3, of which those below `cols` exist): rounded once
template <bool GATED>
__device__ __forceinline__ void few_store(const Few8Args& a, int m, int n, int cols, f32x4 v, const f32x4& u) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if constexpr (GATED) {
            v[r] = f8_unit(v[r], u[r], a.unit, a.limit);
        } else {
            if (a.bias && n + r < cols) v[r] += to_f32(a.bias[n + r]);
        }
    }
    if (!GATED && a.out_float) {
        float* c = (float*)a.C + (size_t)m * a.ldc + n;
        if (n + 4 <= cols) {
            *reinterpret_cast<f8_u32x4_at4*>(c) = __builtin_bit_cast(f8_u32x4, v);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < cols) c[r] = v[r];
        }
    } else {
        bf16* c = (bf16*)a.C + (size_t)m * a.ldc + n;
        if (n + 4 <= cols) {
            *reinterpret_cast<f8_u32x2_at2*>(c) = (f8_u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < cols) c[r] = from_f32<bf16>(v[r]);
        }
    }
}

#define F8_PLACE (16 * 128)  // bytes of a block of a tile in LDS
// Blocks on their way, a wave (12288 x 4096 for one row takes 13.0, 12.8 and 13.4 microseconds with 3, 5 and 7), and tiles whose scales are there or on
// theirs (a power of two): 160 KB of LDS hold them and two times the sums.
#define F8_AHEAD 5
constexpr int few_scales(int xc) { return xc < 3 ? 8 : 4; }
constexpr int few_bytes(int xc, int tm) { return F8_NW * (2 * tm * LLMS_WAVE * 16 + F8_AHEAD * F8_PLACE + few_scales(xc) * 256); }

__device__ __forceinline__ f32x4 few_mfma_8(const f8_u32x4 (&w)[2], const f8_u32x4 (&x)[2], const f32x4& c, uint32_t sw, uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((ext_vector_type(8))) int i32x8;
    const i32x8 a = {(int)w[0][0], (int)w[0][1], (int)w[0][2], (int)w[0][3], (int)w[1][0], (int)w[1][1], (int)w[1][2], (int)w[1][3]};
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sw, 0, (int)sx);
#else
    return c;
#endif
}

template <int XC, int TM, bool GATED, bool XB, bool EIGHT>
__global__ __launch_bounds__(F8_NW * LLMS_WAVE) void gemm_float8_stream_kernel(const Stream8Args s) {
    const Few8Args& a = s.a;
    constexpr int UPT = GATED ? 8 : 16, NI = F8_AHEAD, NS = few_scales(XC);
    static_assert((XC - 1 + NI) / XC + 1 <= NS, "tiles between the one that is multiplied and the last one asked for");
    extern __shared__ __attribute__((aligned(16))) f32x4 sums[];  // [2][F8_NW][TM][64], then the waves' places
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / LLMS_WAVE), lane = tid % LLMS_WAVE;
    const int r16 = lane % 16, g = lane / 16;
    uint8_t* const ring = reinterpret_cast<uint8_t*>(sums + 2 * F8_NW * TM * LLMS_WAVE) + wave * (NI * F8_PLACE + NS * 256);
    uint8_t* const scales = ring + NI * F8_PLACE;
    const int units = GATED ? a.inter : a.N;
    const int share = blockIdx.x, part = blockIdx.y;
    const int u0 = 4 * (share * s.each + min(share, s.more)), u1 = min(units, u0 + 4 * (s.each + (share < s.more ? 1 : 0)));
    const int tiles = (u1 - u0 + UPT - 1) / UPT;
    const int b0 = part * s.part_blocks + wave, blocks = min(a.blocks, (part + 1) * s.part_blocks);  // (the wave's blocks: b0 + 8 c)

    // Two loads: block c of the tile's rows.  In front of a tile's first one the scales of all of the wave's blocks, four to a lane: lanes 16 i .. 16 i + 15
    // those of the first row's 128 (i = 0), the last row's (1), gated: of up's first and last row's (2, 3).  (Rows of others' shares are read as
    // the last of this one; blocks and tiles that do not exist are asked for of buffers without bytes.)
    const int lr = lane / 8, lc = ((lane % 8) ^ (lr / 2)) * 16;  // (of the first 8 rows; of the others the bit of 64 bytes is turned)
    const int s_at = min((b0 & ~3) + F8_NW * (lane % 16), a.s_cols - 4);
    unsigned off0 = 0, off1 = 0;  // of the tile that is asked for
    auto ask = [&](int tile, auto column, int place) {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int c = decltype(column)::n;
        const unsigned here = (unsigned)__builtin_amdgcn_readfirstlane(tile < tiles && b0 + F8_NW * c < blocks ? -1 : 0);
        if constexpr (c == 0) {
            const int first = u0 + tile * UPT;
            const int row0 = min(first + lr, u1 - 1), row1 = GATED ? row0 + a.inter : min(first + 8 + lr, u1 - 1);
            off0 = (unsigned)row0 * (unsigned)a.kp + lc, off1 = (unsigned)row1 * (unsigned)a.kp + (lc ^ 64);
            const int row = min(first + (lane & 16 ? UPT - 1 : 0), u1 - 1) + (GATED && lane >= 32 ? a.inter : 0);
            const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.WS), 0, here, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(scales + tile % NS * 256), 4,
                                                     (unsigned)(row / F8_BLOCK * a.s_cols + s_at), 0, 0, 0);
        }
        const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.W), 0, here, 0x00020000);
        uint8_t* to = ring + place * F8_PLACE;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, off0, (b0 + F8_NW * c) * 128, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(to + 1024), 16, off1, (b0 + F8_NW * c) * 128, 0, 0);
#endif
    };
    // X, then the first blocks: memory answers in the order it is asked, so X is taken to 8 bits while the weights are on their way.  (No load under a
    // condition: each would be waited for by itself.  What does not exist is asked for beyond the end of the buffer, which brings zeros.)
    f8_u32x4 x[XC][TM][2];
    uint32_t sx[XC][TM];
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr unsigned NONE = 0x80000000u;
    const __amdgpu_buffer_rsrc_t from_x = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a.X), 0, s.x_bytes, 0x00020000);
    f8_u32x4 v[XB ? XC : 1][4];
    if constexpr (XB) {
        const unsigned row = (unsigned)(min(r16, a.M - 1) * (int)a.ldx) * 2u + 32u * g;
#pragma unroll
        for (int c = 0; c < XC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = (i / 2) * 64 + (i % 2) * 8, b = b0 + F8_NW * c;
                const bool there = b < blocks && b * 128 + 16 * g + at < a.K;
                v[c][i] = __builtin_bit_cast(f8_u32x4, __builtin_amdgcn_raw_buffer_load_b128(from_x, there ? row + b * 256 + at * 2 : NONE, 0, 0));
            }
    } else {
        const __amdgpu_buffer_rsrc_t from_s = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.XS), 0, s.xs_bytes, 0x00020000);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int m = min(j * 16 + r16, a.M - 1);
            const unsigned row = (unsigned)(m * (int)a.ldx) + 16u * g, row_s = (unsigned)(m * a.ldxs);
#pragma unroll
            for (int c = 0; c < XC; ++c) {
                const int b = b0 + F8_NW * c;
                const unsigned at = b < blocks ? row + b * 128 : NONE;
                x[c][j][0] = __builtin_bit_cast(f8_u32x4, __builtin_amdgcn_raw_buffer_load_b128(from_x, at, 0, 0));
                x[c][j][1] = __builtin_bit_cast(f8_u32x4, __builtin_amdgcn_raw_buffer_load_b128(from_x, at, 64, 0));
                sx[c][j] = __builtin_amdgcn_raw_buffer_load_b8(from_s, b < blocks ? row_s + b : NONE, 0, 0);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    f8_for<NI>([&](auto q) { ask(q.n / XC, Number<decltype(q)::n % XC>(), q.n); });
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (XB) {
#pragma unroll
        for (int c = 0; c < XC; ++c) rounded32(v[c], x[c][0], sx[c][0]);
    }
#endif
    // X as numbers, where the registers suffice.
    constexpr bool KEEP = !EIGHT && XC * TM <= 8;
    Numbers32 kept[KEEP ? XC : 1][TM];
    if constexpr (KEEP) {
#pragma unroll
        for (int c = 0; c < XC; ++c)
#pragma unroll
            for (int j = 0; j < TM; ++j) kept[c][j] = numbers32(x[c][j][0], x[c][j][1], sx[c][j]);
    }
    // Block c of tile `tile`, at `place`, is there once no more is on its way than the `behind` blocks asked for after it.  What was read of LDS before is
    // waited for as well: its place is asked for next, and loads that touch no memory come at once.
    f8_u32x4 w[2];
    uint32_t sw;
    int sw_at = 0;  // of the lane's row among the tile's scales
    auto take = [&](int tile, auto column, int place, auto behind) {
        constexpr int c = decltype(column)::n, B = decltype(behind)::n, n = 2 * B + (c + B) / XC;  // ((c + B) / XC: first blocks among them)
        static_assert(n < 64, "the counter of loads on their way");
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_s_waitcnt((n & 15) | ((n >> 4) << 14) | 0x0070);
        asm volatile("" ::: "memory");
#endif
        const uint8_t* from = ring + place * F8_PLACE;
        w[0] = *reinterpret_cast<const f8_u32x4*>(from + r16 * 128 + (g ^ (r16 / 2)) * 16);
        w[1] = *reinterpret_cast<const f8_u32x4*>(from + r16 * 128 + ((4 + g) ^ (r16 / 2)) * 16);
        if constexpr (c == 0) {
            const int first = u0 + tile * UPT, up = GATED && r16 >= 8 ? a.inter : 0;
            const int other = (min(first + r16 % UPT, u1 - 1) + up) / F8_BLOCK != (first + up) / F8_BLOCK;
            sw_at = tile % NS * 256 + other * 64 + (up ? 128 : 0) + (b0 & 3);
        }
        sw = scales[sw_at + 4 * c];
    };
    int place = 0;  // of the block that is multiplied next
    take(0, Number<0>(), 0, Number<NI - 1>());
    for (int tile = 0; tile < tiles; ++tile) {
        f32x4 acc[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        f8_for<XC>([&](auto column) {
            constexpr int c = decltype(column)::n;
            const f8_u32x4 w8[2] = {w[0], w[1]};
            const uint32_t scale8 = sw;
            Numbers32 wn;
            if constexpr (!EIGHT) wn = numbers32(w[0], w[1], sw);
            const int after = place + 1 < NI ? place + 1 : 0;
            take(tile + (c + 1) / XC, Number<(c + 1) % XC>(), after, Number<NI - 2>());
            ask(tile + (c + NI) / XC, Number<(c + NI) % XC>(), place);  // (the block that was there is in registers)
            place = after;
            if constexpr (EIGHT) {
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[j] = few_mfma_8(w8, x[c][j], acc[j], scale8, sx[c][j]);
                return;
            }
            Numbers32 xn[TM];
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                if constexpr (KEEP) {
                    xn[j] = kept[c][j];
                } else {
                    asm volatile("" : "+v"(x[c][j][0]), "+v"(x[c][j][1]));  // (or all of X would be kept as numbers, in twice the registers)
                    xn[j] = numbers32(x[c][j][0], x[c][j][1], sx[c][j]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wn.v[k], xn[j].v[k], acc[j], 0, 0, 0);
        });
        f32x4* meet = sums + (tile & 1) * F8_NW * TM * LLMS_WAVE;  // [F8_NW][TM][64]
#pragma unroll
        for (int j = 0; j < TM; ++j) meet[(wave * TM + j) * LLMS_WAVE + lane] = acc[j];
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_s_waitcnt(0xc07f);  // (LDS only: the next blocks stay on their way)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#endif
        // a thread adds up a lane's 4 sums (GATED: of 4 gates, and of the same units' ups 32 lanes further on)
        constexpr int LANES = GATED ? 32 : 64;
        if (tid < TM * LANES) {
            const int l = tid % LANES, j = tid / LANES, m = j * 16 + l % 16, n = u0 + tile * UPT + 4 * (l / 16);
            f32x4 v = {0.f, 0.f, 0.f, 0.f}, u = v;
#pragma unroll
            for (int k = 0; k < F8_NW; ++k) {
                v += meet[(k * TM + j) * LLMS_WAVE + l];
                if constexpr (GATED) u += meet[(k * TM + j) * LLMS_WAVE + l + 32];
            }
            if (m < a.M && n < u1) {
                if (s.sums) {
                    float* to = s.sums + ((size_t)part * a.M + m) * s.ld + n;
                    *reinterpret_cast<f32x4*>(to) = v;
                    if constexpr (GATED) *reinterpret_cast<f32x4*>(to + s.up_at) = u;
                } else {
                    few_store<GATED>(a, m, n, u1, v, u);
                }
            }
        }
    }
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_s_waitcnt(0);  // (no load may find the workgroup gone)
#endif
}

// The parts' sums, added up in their order: a thread four units of a row.
template <bool GATED>
__global__ __launch_bounds__(256) void gemm_float8_join_kernel(const Stream8Args s) {
    const Few8Args& a = s.a;
    const int at = blockIdx.x * 256 + threadIdx.x, m = at / s.quads, n = 4 * (at - m * s.quads), units = GATED ? a.inter : a.N;
    if (m >= a.M) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f}, u = v;
    for (int p = 0; p < s.parts; ++p) {
        const float* from = s.sums + ((size_t)p * a.M + m) * s.ld + n;
        v += *reinterpret_cast<const f32x4*>(from);
        if constexpr (GATED) u += *reinterpret_cast<const f32x4*>(from + s.up_at);
    }
    few_store<GATED>(a, m, n, units, v, u);
}

template <int XC, int TM, bool GATED, bool XB, bool EIGHT>
static int stream_launch(const Stream8Args& s, int shares, hipStream_t stream) {
    constexpr int bytes = few_bytes(XC, TM);
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    auto kernel = gemm_float8_stream_kernel<XC, TM, GATED, XB, EIGHT>;
    static bool set[64] = {};
    if (const int failed = f8_raise_lds(reinterpret_cast<const void*>(kernel), bytes, set)) return failed;
    kernel<<<dim3(shares, s.parts), F8_NW * LLMS_WAVE, bytes, stream>>>(s);
    if (s.sums) gemm_float8_join_kernel<GATED><<<(s.quads * s.a.M + 255) / 256, 256, 0, stream>>>(s);
    LLMS_LAUNCH_CHECK();
}

template <int XC, int TM, bool GATED>
static int stream_go(Stream8Args& s, bool x_bf16, int cus, hipStream_t stream) {
    const int shares = min(s.quads, max(1, cus / s.parts));
    s.each = s.quads / shares, s.more = s.quads % shares;
    if constexpr (TM == 1 && XC <= 4)
        if (x_bf16) return stream_launch<XC, TM, GATED, true, false>(s, shares, stream);
    LLMS_REQUIRE(!x_bf16, "gemm_float8_few: more rows or columns in bfloat16 than are taken to 8 bits on the way in");
    if constexpr (TM > 1)
        if (!s.a.out_float) return stream_launch<XC, TM, GATED, false, true>(s, shares, stream);
    if constexpr (TM == 1 || !GATED) return stream_launch<XC, TM, GATED, false, false>(s, shares, stream);
    LLMS_REQUIRE(false, "gemm_float8_few: gated results are bfloat16");
}

// (blocks of K a wave: as many as leave X and the products room in 256 registers)
template <bool GATED>
static int stream_rows(Stream8Args& s, int row_blocks, bool x_bf16, int cus, hipStream_t st) {
    const int xc = (s.part_blocks + F8_NW - 1) / F8_NW;
#define GO(XC, TM) \
    if (xc <= XC) return stream_go<XC, TM, GATED>(s, x_bf16, cus, st)
    if (row_blocks == 1) {
        GO(1, 1);
        GO(2, 1);
        GO(3, 1);
        GO(4, 1);
        GO(6, 1);
        GO(8, 1);
        GO(11, 1);
        GO(14, 1);
    } else if (row_blocks == 2) {
        GO(1, 2);
        GO(2, 2);
        GO(3, 2);
        GO(4, 2);
        GO(6, 2);
        GO(8, 2);
    } else {
        GO(1, 4);
        GO(2, 4);
        GO(3, 4);
        GO(4, 4);
    }
#undef GO
    LLMS_REQUIRE(false, "gemm_float8_few: no such share of K");
}

template <int EPI, bool XB>
static int few_groups(const Few8Args& a, int groups, hipStream_t stream) {
    constexpr int TN = 2, TM = 1;
    const int rows = EPI == G8_GATED ? 32 * ((a.inter + 15) / 16) : a.N;
    gemm_float8_few_kernel<TN, TM, EPI, XB><<<dim3((rows + 16 * TN - 1) / (16 * TN), groups), F8_NW * LLMS_WAVE, F8_NW * TN * TM * LLMS_WAVE * 16, stream>>>(a);
    LLMS_LAUNCH_CHECK();
}

// epilogue: 0 bfloat16, 1 float, 2 gated.  x_bf16: X is bfloat16 with K columns (a multiple of 8, rows on 16 bytes).  Without seg, up to 64 rows:
// row_blocks (1, 2 or 4) of 16; `parts` of K, whose sums go to `sums` [parts][m][ld] where there are several (ld: n up to a multiple of 4;
// gated: gate and up each up to one).  With seg, groups of rows (a weight each), of any number.
extern "C" int llms_gemm_float8_few(int epilogue, int x_bf16, int row_blocks, void* c, long ldc, const void* x, long ldx, const void* xs, int ldxs,
                                    const void* w, const void* ws, int s_cols, const void* bias, int m, int n, int k, int unit, float limit,
                                    const int* seg, int groups, long w_stride, long ws_stride, int parts, void* sums, int cus, void* stream) {
    const long kp = F8_BLOCK * (((long)k + F8_BLOCK - 1) / F8_BLOCK);
    LLMS_REQUIRE(m > 0 && n > 0 && k > 0 && cus > 0 && n * kp < (1l << 32) - (1 << 23), "gemm_float8_few sizes");
    LLMS_REQUIRE(seg ? groups > 0 && groups < 65536 : m <= 16 * row_blocks && parts > 0 && (parts == 1 || sums), "gemm_float8_few rows");
    LLMS_REQUIRE(epilogue < G8_GATED || n % 2 == 0, "gemm_float8_few: gate and up have the same rows");
    Few8Args a = {};
    a.X = x, a.XS = (const uint8_t*)xs, a.W = (const uint8_t*)w, a.WS = (const uint8_t*)ws, a.bias = (const bf16*)bias, a.C = c;
    a.ldx = ldx, a.ldc = ldc, a.ldxs = ldxs, a.s_cols = s_cols, a.M = m, a.N = n, a.K = k;
    a.blocks = (int)(kp / F8_BLOCK), a.kp = (int)kp;
    a.inter = epilogue == G8_GATED ? n / 2 : 0, a.unit = unit, a.limit = limit, a.out_float = epilogue == G8_FLOAT;
    a.seg = seg, a.w_stride = w_stride, a.ws_stride = ws_stride;
    hipStream_t st = (hipStream_t)stream;
    if (!seg) {
        Stream8Args s = {};
        const int units = epilogue == G8_GATED ? a.inter : n;
        s.a = a, s.quads = (units + 3) / 4, s.parts = parts, s.part_blocks = (a.blocks + parts - 1) / parts;
        s.sums = parts > 1 ? (float*)sums : nullptr, s.up_at = 4 * s.quads, s.ld = (epilogue == G8_GATED ? 8 : 4) * s.quads;
        LLMS_REQUIRE(ldx < (1 << 23) && ldxs < (1 << 23), "gemm_float8_few: rows too far apart");
        s.x_bytes = (unsigned)(((m - 1) * ldx + (x_bf16 ? k : kp)) * (x_bf16 ? 2 : 1)), s.xs_bytes = (unsigned)((m - 1) * ldxs + s_cols);
        return epilogue == G8_GATED ? stream_rows<true>(s, row_blocks, x_bf16, cus, st) : stream_rows<false>(s, row_blocks, x_bf16, cus, st);
    }
#define GO(EPI) return x_bf16 ? few_groups<EPI, true>(a, groups, st) : few_groups<EPI, false>(a, groups, st)
    if (epilogue == G8_BF16) GO(G8_BF16);
    if (epilogue == G8_FLOAT) GO(G8_FLOAT);
    GO(G8_GATED);
#undef GO
}
