// mvh_fp8.hip -- weights in 8-bit floating point (e4m3) with a float scale per
// 128 x 128 block: quantisation, products, and the gated feed-forward block.
//
//   y[b][r] = sum_k sa[b][k] sw[r / 128][k] sum_{i in block k} qa[b][i] qw[r][i]
// with x row b held as e4m3 codes qa and a scale sa per 128 columns.
//
// The inner sums run on the fp16 matrix pipe, which codes (4 bits each) enter
// exactly.  The 8-bit pipe has twice its rate, but aligns eight products at a time
// and cuts each 13 bits below the largest: sums of 128 were off by 1.4e-5 of
// themselves against 64 bits, 40 times what they are here.
#include "mvh_kernels.hpp"

namespace mvh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlk = 128;
constexpr float kTop = 448.0f;            // largest e4m3 value
constexpr float kLeast = 0x1p-126f;       // scales below are no normal numbers: the block is held as zeros

// 32 codes as fp16
struct Codes32 {
    half8 h[4];
};
__device__ __forceinline__ half8 to_half8(uint32_t a, uint32_t b) {
    const half2v h0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), h1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const half2v h2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), h3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return half8{h0.x, h0.y, h1.x, h1.y, h2.x, h2.y, h3.x, h3.y};
}
__device__ __forceinline__ Codes32 widen(uint4 a, uint4 b) {
    return {{to_half8(a.x, a.y), to_half8(a.z, a.w), to_half8(b.x, b.y), to_half8(b.z, b.w)}};
}
// 16 x 16 sums of 128 products: a = rows, b = columns; lane (n, j) holds 32 codes
// of row / column n, the same ones of each, and gets column n of rows 4 j ..
__device__ __forceinline__ f32x4 dot128(const Codes32& a, const Codes32& b) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h[i], b.h[i], c, 0, 0, 0);
    return c;
}

// The scale of a block whose largest |x| has these bits (NaN above infinity above
// all numbers, so either reaches the scale), and its inverse
__device__ __forceinline__ float scale_of(uint32_t top) {
    const float s = __fdiv_rn(__uint_as_float(top), kTop);
    return s < kLeast ? 0.0f : s;
}
__device__ __forceinline__ float inverse_of(float s) { return s == 0.0f ? 0.0f : __fdiv_rn(1.0f, s); }
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t top4(float4 v) {
    return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
}
__device__ __forceinline__ uint32_t codes4(float4 v, float inv) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v.x * inv, v.y * inv, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v.z * inv, v.w * inv, w, true));
}
// max over aligned groups of 32 lanes
__device__ __forceinline__ uint32_t half_max(uint32_t m) {
    auto up = [](uint32_t a, int b) { return max(a, static_cast<uint32_t>(b)); };
    m = up(m, dpp_mov<0xb1>(static_cast<int>(m)));
    m = up(m, dpp_mov<0x4e>(static_cast<int>(m)));
    m = up(m, dpp_mov<0x141>(static_cast<int>(m)));
    m = up(m, dpp_mov<0x140>(static_cast<int>(m)));
    return up(m, swz_xor<16>(static_cast<int>(m)));
}

// x [rows][cols] -> codes (rows `pitch` apart, columns cols .. pitch zero up to the
// last block's end) and scales[row * row_step + block * block_step]: 32 lanes a
// block, 16 bytes each.
__global__ __launch_bounds__(256) void quantize_rows_kernel(const float* __restrict__ x, int cols, int blocks, size_t items,
                                                            uint8_t* __restrict__ codes, size_t pitch,
                                                            float* __restrict__ scales, size_t row_step, size_t block_step) {
    const int lane = threadIdx.x & 31;
    const size_t item = static_cast<size_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (item >= items) return;
    const size_t row = item / blocks;
    const int kb = static_cast<int>(item % blocks), at = kb * kBlk + lane * 4;
    const float4 v = at < cols ? *reinterpret_cast<const float4*>(x + row * cols + at) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float s = scale_of(half_max(top4(v)));
    const uint32_t c = codes4(v, inverse_of(s));
    if (static_cast<size_t>(at) < pitch) *reinterpret_cast<uint32_t*>(codes + row * pitch + at) = c;
    if (lane == 0) scales[row * row_step + kb * block_step] = s;
}

// The same with a scale per 128 x 128: a workgroup a block
__global__ __launch_bounds__(256) void quantize_tiles_kernel(const float* __restrict__ x, size_t rows, int cols, int blocks,
                                                             uint8_t* __restrict__ codes, float* __restrict__ scales) {
    __shared__ uint32_t s_top[4];
    const int kb = static_cast<int>(blockIdx.x % blocks);
    const size_t rb = blockIdx.x / blocks, r0 = rb * kBlk + (threadIdx.x >> 5);
    const int at = kb * kBlk + (threadIdx.x & 31) * 4;
    float4 v[16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const size_t r = r0 + 8 * i;
        v[i] = r < rows && at < cols ? *reinterpret_cast<const float4*>(x + r * cols + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(top, top4(v[i]));
    }
    top = half_max(top);
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
    const float s = scale_of(max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]))), inv = inverse_of(s);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const size_t r = r0 + 8 * i;
        if (r < rows && at < cols) *reinterpret_cast<uint32_t*>(codes + r * cols + at) = codes4(v[i], inv);
    }
    if (threadIdx.x == 0) scales[rb * blocks + kb] = s;
}

struct Fp8Args {
    const uint8_t* w[2];   // codes [N][K]
    const float* ws[2];    // scales [ceil(N / 128)][blocks]
    const uint8_t* xq;     // codes [M][128 blocks], zeros behind column K
    const float* xs;       // scales [blocks][M]
    float* y;              // [M][N]
    int N, K, M, blocks, gate;
};

__device__ __forceinline__ float gated(float g, float u, int gate) {
    const float a = gate == kGateSilu ? __fdiv_rn(g, 1.0f + expf(-g)) : 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
    return a * u;
}

// One workgroup: 16 rows of the weights, 16 TT tokens, its waves the blocks of K
// in turn.
template <int MATS, int TT, int W>
__global__ __launch_bounds__(64 * W) void fp8_rows_kernel(Fp8Args a) {
    __shared__ float s_y[W][MATS][TT][16][17];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int r0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * TT, last16 = a.K / 16 - 1;
    const size_t pitch = static_cast<size_t>(a.blocks) * kBlk;
    const uint8_t* wp[MATS];
    const float* sp[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        wp[m] = a.w[m] + static_cast<size_t>(min(r0 + n, a.N - 1)) * a.K;
        sp[m] = a.ws[m] + static_cast<size_t>(r0 / kBlk) * a.blocks;
    }
    f32x4 acc[MATS][TT];
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < a.blocks; kb += W) {
        // a last block that is short: columns of the row again, against zeros
        const size_t c0 = 16 * static_cast<size_t>(min(kb * 8 + j, last16)), c1 = 16 * static_cast<size_t>(min(kb * 8 + 4 + j, last16));
        Codes32 w[MATS];
        float ws[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            w[m] = widen(ld_global16(wp[m] + c0), ld_global16(wp[m] + c1));
            ws[m] = sp[m][kb];
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int tok = min(t0 + 16 * t + n, a.M - 1);
            const uint8_t* xp = a.xq + tok * pitch + kb * kBlk + 16 * j;
            const Codes32 x = widen(ld_global16(xp), ld_global16(xp + 64));
            const float xs = a.xs[static_cast<size_t>(kb) * a.M + tok];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                const f32x4 c = dot128(w[m], x);
                const float s = xs * ws[m];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][t][i] = fmaf(s, c[i], acc[m][t][i]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_y[wave][m][t][n][4 * j + i] = acc[m][t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * TT; e += 64 * W) {
        const int t = e >> 8, tok = (e >> 4) & 15, r = e & 15;
        float v[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            v[m] = s_y[0][m][t][tok][r];
#pragma unroll
            for (int k = 1; k < W; ++k) v[m] += s_y[k][m][t][tok][r];
        }
        const int token = t0 + 16 * t + tok;
        if (token < a.M && r0 + r < a.N)
            a.y[static_cast<size_t>(token) * a.N + r0 + r] = MATS == 2 ? gated(v[0], v[MATS - 1], a.gate) : v[0];
    }
}

// TM tokens x TN rows of the weights (with two matrices TN / 2 of each), four
// waves of half the tokens and half the rows each; a step is one block of 128
// columns.  The codes go from memory to LDS as they are, one step ahead, and are
// widened behind it: as fp16 they would take twice the LDS reads, which at 64 x 64
// a wave are half of the matrix pipe's time already.
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

template <int TM, int TN>
struct Step {  // rows of 128 bytes, their 16-byte chunks turned by the row: 16 rows' reads fall in different banks
    uint8_t x[TM * kBlk], w[TN * kBlk];
};
__device__ __forceinline__ int turn(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ Codes32 codes_at(const uint8_t* rows, int row, int j) {
    const uint8_t* r = rows + row * kBlk;
    return widen(*reinterpret_cast<const uint4*>(r + ((j ^ turn(row)) * 16)), *reinterpret_cast<const uint4*>(r + (((j + 4) ^ turn(row)) * 16)));
}

template <int MATS, int TM, int TN>
__global__ __launch_bounds__(256, 2) void fp8_tile_kernel(Fp8Args a) {
    constexpr int WM = TM / 2, WN = TN / 2, XT = WM / 16, WT = WN / 16, PER = TN / MATS;  // PER: rows of a matrix
    __shared__ __align__(16) Step<TM, TN> s0, s1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    // tiles in eight runs, one per XCD (workgroups go to them in turn), tokens first: an XCD's L2 then holds few rows of the weights at a time
    const int tiles_m = (a.M + TM - 1) / TM, tiles = tiles_m * ((a.N + PER - 1) / PER);
    const int id = blockIdx.x, share = tiles / 8, more = tiles % 8, xcd = id & 7;
    const int tile = xcd * share + min(xcd, more) + (id >> 3);
    const int t0 = tile % tiles_m * TM, r0 = tile / tiles_m * PER;
    const size_t pitch = static_cast<size_t>(a.blocks) * kBlk;
    const uint32_t last = static_cast<uint32_t>(a.K - 16);

    // eight rows of 128 bytes an instruction
    constexpr int XI = TM / 32, WI = TN / 32;
    uint32_t xo[XI], wo[WI];
    const int in = lane >> 3, c = lane & 7;
    const uint8_t* const xb = a.xq + static_cast<size_t>(t0) * pitch;
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int row = (i * 4 + wave) * 8 + in;
        xo[i] = static_cast<uint32_t>(min(row, a.M - 1 - t0)) * static_cast<uint32_t>(pitch) + ((c ^ turn(row)) * 16);
    }
    uint32_t wc[WI];
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int row = (i * 4 + wave) * 8 + in;
        wo[i] = static_cast<uint32_t>(min(row % PER, a.N - 1 - r0)) * static_cast<uint32_t>(a.K);
        wc[i] = (c ^ turn(row)) * 16;
    }
    auto load = [&](Step<TM, TN>& s, int kb) {
#pragma unroll
        for (int i = 0; i < XI; ++i)
            __builtin_amdgcn_global_load_lds((global_void*)(xb + (xo[i] + static_cast<uint32_t>(kb) * kBlk)),
                                             (lds_void*)(s.x + (i * 4 + wave) * 1024), 16, 0, 0);
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int m = MATS == 2 ? (i * 4 + wave) * 8 / PER : 0;
            const uint8_t* const wb = (m ? a.w[1] : a.w[0]) + static_cast<size_t>(r0) * a.K;
            // a last block that is short: columns of the row again, against zeros
            __builtin_amdgcn_global_load_lds((global_void*)(wb + (wo[i] + min(static_cast<uint32_t>(kb) * kBlk + wc[i], last))),
                                             (lds_void*)(s.w + (i * 4 + wave) * 1024), 16, 0, 0);
        }
    };
    const float* xs[XT];
#pragma unroll
    for (int t = 0; t < XT; ++t) xs[t] = a.xs + min(t0 + wm * WM + 16 * t + n, a.M - 1);
    float xn[XT], wsn[MATS];
    auto scales = [&](int kb) {
#pragma unroll
        for (int t = 0; t < XT; ++t) xn[t] = xs[t][static_cast<size_t>(kb) * a.M];
#pragma unroll
        for (int m = 0; m < MATS; ++m) wsn[m] = a.ws[m][static_cast<size_t>(r0 / kBlk) * a.blocks + kb];
    };

    f32x4 acc[WT][XT];
#pragma unroll
    for (int w = 0; w < WT; ++w)
#pragma unroll
        for (int t = 0; t < XT; ++t) acc[w][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto step = [&](const Step<TM, TN>& s, Step<TM, TN>& next, int kb) {
        float sc[MATS][XT];
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int t = 0; t < XT; ++t) sc[m][t] = xn[t] * wsn[m];
        __syncthreads();
        if (kb + 1 < a.blocks) {
            load(next, kb + 1);
            scales(kb + 1);
        }
        Codes32 x[XT];
#pragma unroll
        for (int t = 0; t < XT; ++t) x[t] = codes_at(s.x, wm * WM + 16 * t + n, j);
#pragma unroll
        for (int w = 0; w < WT; ++w) {
            const int m = MATS == 2 ? w / (WT / 2) : 0;
            const int row = MATS == 2 ? m * PER + wn * (WN / 2) + 16 * (w % (WT / 2)) : wn * WN + 16 * w;
            const Codes32 v = codes_at(s.w, row + n, j);
#pragma unroll
            for (int t = 0; t < XT; ++t) {
                const f32x4 d = dot128(v, x[t]);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[w][t][i] = fmaf(sc[m][t], d[i], acc[w][t][i]);
            }
        }
    };
    load(s0, 0);
    scales(0);
    for (int kb = 0; kb < a.blocks; kb += 2) {
        step(s0, s1, kb);
        if (kb + 1 < a.blocks) step(s1, s0, kb + 1);
    }

    const bool vec = a.N % 4 == 0;
#pragma unroll
    for (int t = 0; t < XT; ++t) {
        const int token = t0 + wm * WM + 16 * t + n;
        if (token >= a.M) continue;
#pragma unroll
        for (int w = 0; w < WT / MATS; ++w) {
            const int r = r0 + wn * (WN / MATS) + 16 * w + 4 * j;
            f32x4 v = acc[w][t];
            if constexpr (MATS == 2)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = gated(v[i], acc[w + WT / 2][t][i], a.gate);
            float* y = a.y + static_cast<size_t>(token) * a.N + r;
            if (vec && r + 3 < a.N) *reinterpret_cast<f32x4*>(y) = v;
            else
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r + i < a.N) y[i] = v[i];
        }
    }
}

template <int MATS>
void launch_tile(const Fp8Args& a, hipStream_t st) {
    const int big = ((a.M + 127) / 128) * ((a.N * MATS + 127) / 128);
    if (big >= 200) {
        fp8_tile_kernel<MATS, 128, 128><<<dim3(static_cast<unsigned>((a.M + 127) / 128) * ((a.N + 128 / MATS - 1) / (128 / MATS))), 256, 0, st>>>(a);
    } else {
        fp8_tile_kernel<MATS, 64, 64><<<dim3(static_cast<unsigned>((a.M + 63) / 64) * ((a.N + 64 / MATS - 1) / (64 / MATS))), 256, 0, st>>>(a);
    }
}

}  // namespace

size_t fp8_scratch(size_t K, size_t M) {
    const size_t blocks = (K + kBlk - 1) / kBlk;
    return M * blocks * (kBlk + 4);
}

hipError_t launch_quantize_fp8(const float* x, size_t rows, size_t cols, size_t block_rows, uint8_t* codes, float* scales,
                               hipStream_t st) {
    const int blocks = static_cast<int>((cols + kBlk - 1) / kBlk);
    if (block_rows == 1) {
        const size_t items = rows * blocks;
        quantize_rows_kernel<<<dim3(static_cast<unsigned>((items + 7) / 8)), 256, 0, st>>>(
            x, static_cast<int>(cols), blocks, items, codes, cols, scales, blocks, 1);
    } else {
        const size_t tiles = (rows + kBlk - 1) / kBlk * blocks;
        quantize_tiles_kernel<<<dim3(static_cast<unsigned>(tiles)), 256, 0, st>>>(x, rows, static_cast<int>(cols), blocks, codes,
                                                                                  scales);
    }
    return hipGetLastError();
}

hipError_t launch_fp8(const uint8_t* w, const uint8_t* w2, int gate, const float* x, float* y, size_t N, size_t K, size_t M,
                      void* scratch, hipStream_t st) {
    const size_t blocks = (K + kBlk - 1) / kBlk, items = M * blocks;
    Fp8Args a{};
    a.N = static_cast<int>(N), a.K = static_cast<int>(K), a.M = static_cast<int>(M), a.blocks = static_cast<int>(blocks);
    a.gate = gate;
    a.w[0] = w, a.w[1] = w2;
    a.ws[0] = reinterpret_cast<const float*>(w + N * K);
    a.ws[1] = w2 ? reinterpret_cast<const float*>(w2 + N * K) : nullptr;
    auto* xq = static_cast<uint8_t*>(scratch);
    auto* xs = reinterpret_cast<float*>(xq + M * blocks * kBlk);
    a.xq = xq, a.xs = xs, a.y = y;
    quantize_rows_kernel<<<dim3(static_cast<unsigned>((items + 7) / 8)), 256, 0, st>>>(
        x, a.K, a.blocks, items, xq, blocks * kBlk, xs, 1, M);
    if (M > 64) {
        if (w2) launch_tile<2>(a, st);
        else launch_tile<1>(a, st);
        return hipGetLastError();
    }
    const dim3 grid(static_cast<unsigned>((N + 15) / 16), static_cast<unsigned>((M + 15) / 16));
    if (w2) fp8_rows_kernel<2, 1, 4><<<grid, 256, 0, st>>>(a);
    else fp8_rows_kernel<1, 1, 4><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace mvh
