// mvh_attn_q4.hip -- attention over a paged KV cache held in 4 bits (layout
// and format: mvh_kv4.hpp), of one token or a chunk of tokens.
//
//   y_t = log2(e) / sqrt(hd) * q.K_t,  out = sum_t 2^(y_t - m) V_t / sum_t 2^(y_t - m)
// over rows t = 0 .. the token's position, in one pass with a running m.  Per
// block of 32 channels K_t = c + s (n - 8), so
//   q.K_t       = sum_b s_tb (sum_i q_i (n_ti - 8)) + c_tb sum_i q_i,
//   sum p_t V_t = sum_t (p_t s_tb) (n_t - 8) + sum_t p_t c_tb :
// n - 8 is exact in fp16, so the products run on the fp16 matrix pipe with the
// codes as they are; q and p s are split into two fp16 (22 bits, where one fp16
// would leave 11), sums are fp32.
#include "mvh_kernels.hpp"
#include "mvh_kv4.hpp"

#include <numeric>
#include <type_traits>

namespace mvh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
template <int NB>
struct NQuad {  // registers that hold a number per block in four lanes
    static constexpr int value = (NB + 3) / 4;
};

struct Q4Args {
    const void* const* pt_k;
    const void* const* pt_v;
    const float* q;
    float* out;
    float* part;  // [row][split][hd], then [row][split][2]: sums and (m, l); null with one split
    const int* d_pos;
    size_t q_pitch;
    int pos, n_tokens, n_head, group, kv_dim, hd;
    int chunk;  // 32-row steps a split takes; 0: the rows' steps shared out evenly
    Kv4Map map;
};

constexpr float kLowest = -1.0e12f;  // m before the first row, below any score of a scaled query: finite, so that 2^(-inf - m) is 0
constexpr float kLog2e = 1.44269504088896340736f;
// Weights are 2^(y - m + kLift), and m follows the maximum only when that is
// kSlack ahead (the sums are rescaled seldom, the decision is each row's own): at
// most 2^14.  fp16 keeps 22 bits of such a weight in two parts down to 2^-12 of
// the largest, and 2^-35 of the largest below.
//
// p s keeps that range only where a block's steps are near 1.  So a block's sums
// are held times a power of two u, by the largest step that the query row has
// seen there (unit_of): 1 while that is in [2^-7, 2), else what brings it to [1/2,
// 1); it falls, and the sums with it, when a step times u reaches 2.  u >= 1
// scales the steps, exactly; blocks with u < 1 (a step of 2 .. 512) form p s u in
// 32 bits and split it.  p s u is below 2^15, and p s off by 2^-22 of itself or
// 2^-28 of the largest weight times the block's largest step (2^-35 where that is
// not in [2^-7, 1)), whatever other blocks hold.  A wave's first step looks whether
// all its blocks start with u = 1; while they stay there, the usual case, steps
// are taken as they are.  256 tokens at
// 16000, 8 kv heads of 128: 180 us, with values of size 0.01 191, with a row of 200 in
// one block of each head 195; one u for the head was 177.
//
// The exponent of a weight is y_scale s - y_scale m + kLift, the second product
// rounded once for all of a step's rows (and for the join); where it is beyond
// kFar, and that rounding a large factor, m is taken off the scores first.  So is
// the m of a query row that has seen nothing yet.
constexpr float kLift = 10.0f, kSlack = 4.0f, kFar = 1048576.0f;
constexpr uint32_t kUnitOne = 0x3c00u, kUnitFirst = 30u << 10;  // 1, and 2^15: before any step
constexpr uint32_t kUsualBits = 0x60006000u, kWideBits = 0x40004000u;  // of a step >= 2^-7, >= 2 (or NaN), in either half
constexpr int kWaves = 4;
constexpr int kTile = 16;  // query rows of a workgroup

__device__ __forceinline__ int steps_of(const Kv4Map& map, int lim) { return map.group_of(lim) / 4 + 1; }
// a split's steps: whole turns of the workgroup's waves, by two steps at a time
__device__ __forceinline__ int split_chunk(const Q4Args& a, int pos, int n_split) {
    if (a.chunk) return a.chunk;
    const int per = (steps_of(a.map, pos + a.n_tokens - 1) + n_split - 1) / n_split;
    return (per + 2 * kWaves - 1) / (2 * kWaves) * (2 * kWaves);
}

__device__ __forceinline__ uint32_t rows_max_bits(uint32_t v) {
    auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// u of a block whose largest step has these bits (NaN: as the largest step there is)
__device__ __forceinline__ uint32_t unit_of(uint32_t step) {
    const uint32_t e = min(step >> 10, 24u);
    return e >= 8 && e < 16 ? kUnitOne : (29 - e) << 10;
}
// a step times u that is 2 or more, or NaN, shows in bit 14 of its half
__device__ __forceinline__ uint32_t reaches_2(uint32_t steps, half2v u) { return as_u32(as_half2(steps) * u) & kWideBits; }
__device__ __forceinline__ half2v both(uint32_t u) { return as_half2(u | (u << 16)); }
__device__ __forceinline__ bool below_1(half2v u) { return (as_u32(u) & 0xffffu) < kUnitOne; }
__device__ __forceinline__ float unit_f(half2v u) { return static_cast<float>(u.x); }
__device__ __forceinline__ float unit_inverse(half2v u) {  // of a power of two
    return __uint_as_float((254u << 23) - __float_as_uint(unit_f(u)));
}
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t max_half(uint32_t a) { return max(a & 0xffffu, a >> 16); }

// Loads at a base that is the same in every lane plus a 32-bit offset: the base
// stays in scalar registers.
__device__ __forceinline__ uint2 ld8_at(const uint8_t* base, uint32_t off) {
    const auto* b = (const __attribute__((address_space(1))) uint8_t*)(reinterpret_cast<uintptr_t>(base));
    const u32x2 v = *(const __attribute__((address_space(1))) u32x2*)(b + off);
    return make_uint2(v.x, v.y);
}
__device__ __forceinline__ uint32_t ld4_at(const uint8_t* base, uint32_t off) {
    const auto* b = (const __attribute__((address_space(1))) uint8_t*)(reinterpret_cast<uintptr_t>(base));
    return *(const __attribute__((address_space(1))) uint32_t*)(b + off);
}
__device__ __forceinline__ u32x4 ld16_at(const uint8_t* base, uint32_t off) {
    const auto* b = (const __attribute__((address_space(1))) uint8_t*)(reinterpret_cast<uintptr_t>(base));
    return *(const __attribute__((address_space(1))) u32x4*)(b + off);
}
// An entry of a page table through the scalar cache (page: the same in every lane)
__device__ __forceinline__ const uint8_t* page_at(const void* const* pt, int page) {
    typedef const __attribute__((address_space(4))) uint64_t* entry;
    return reinterpret_cast<const uint8_t*>(*reinterpret_cast<entry>(reinterpret_cast<uintptr_t>(pt + page)));
}

// a times (high + low) + c, the low parts first
__device__ __forceinline__ f32x4 mfma2(u32x4 a, u32x4 high, u32x4 low, f32x4 c) {
    const half8 m = __builtin_bit_cast(half8, a);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(m, __builtin_bit_cast(half8, low), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(m, __builtin_bit_cast(half8, high), c, 0, 0, 0);
}
// p - h (exact where h is p rounded, or 0): the conversion inside the addition
__device__ __forceinline__ float less(float p, _Float16 h, float minus1) { return fmaf(static_cast<float>(h), minus1, p); }

// Two weights (in two parts each) times their steps, in two parts: the product rounded, and what that lost plus lo s
__device__ __forceinline__ void times_steps(half2v hi, half2v lo, half2v s, uint32_t& h, uint32_t& l) {
    const half2v t = hi * s;
    half2v w = __builtin_elementwise_fma(hi, s, -t);
    w = __builtin_elementwise_fma(lo, s, w);
    h = as_u32(t);
    l = as_u32(w);
}
// Two weights times their steps and u in 32 bits, in two parts
__device__ __forceinline__ void times_steps(float p, float q, half2v s, float u, float minus1, uint32_t& h, uint32_t& l) {
    const float x = p * static_cast<float>(s.x) * u, y = q * static_cast<float>(s.y) * u;
    const half2v t = pk_half(x, y);
    h = as_u32(t);
    l = as_u32(pk_half(less(x, t.x, minus1), less(y, t.y, minus1)));
}

// A workgroup's result for channel d of query row `row`: the output, or the split's part of it
__device__ __forceinline__ void write_sum(const Q4Args& a, int kh, int row, int d, int hd, int n_split, float sum, float l, float top) {
    const size_t out_row = static_cast<size_t>(row / a.group) * a.n_head + kh * a.group + row % a.group;
    if (!a.part) {
        a.out[out_row * hd + d] = __fdiv_rn(sum, l);
        return;
    }
    const size_t at = out_row * n_split + blockIdx.z;
    a.part[at * hd + d] = sum;
    if (d == 0) {
        float* ml = a.part + static_cast<size_t>(a.n_tokens) * a.n_head * n_split * hd + 2 * at;
        ml[0] = top;
        ml[1] = l;
    }
}

// One workgroup: 16 query rows (row = token * group + head of the kv head) of
// kv head x, tile y, split z.  Its four waves take 32-row steps in turn, each
// with a running maximum of its own, and join through LDS.
//
// The matrix pipe's 16 columns are the query rows; the high and the low parts
// go through it one after the other.  Scores come transposed (rows of the operand = cache rows), so a lane
// then holds p of 8 consecutive cache rows of one query row: with the cache
// rows in that order in V's words too, p is the next product's operand as it
// is.  sum p c and sum p are one more product whose operand rows are the
// blocks' c, and ones.  64 query rows on 8 kv heads of 128 at position 1500: 13.5
// us, 8 rows at 30000: 19.0 (2.1 TB/s).  Neither pipe is a bound (VALU 20 and 40 %
// busy, matrix pipe 3 and 11 %): two waves per SIMD wait for their loads and for
// each other's turns, at the start most of all (a token at 100: 5.8 us).
//
// PART: heads that do not fill NB whole blocks.  A head's channels lie in the
// blocks from its first one on, with q zero at the others' channels of these
// (6 heads of 48 at position 1500: 9.6 us, 64 tokens there 12.1; on the kernel
// for heads of more than 8 blocks 35.3 and 192).
template <int NB, bool UNI, bool PART>
__global__ __launch_bounds__(64 * kWaves, NB > 4 ? 1 : 2) void attn_q4_kernel(Q4Args a) {
    constexpr int HD = 32 * NB, PITCH = HD + 4;
    __shared__ float s_o[kWaves][kTile][PITCH];
    __shared__ float s_c[kWaves][kTile][12];  // [0..NB) sum p c of the blocks, [NB] sum p
    __shared__ float s_m[kWaves][kTile];
    __shared__ uint32_t s_unit[kWaves][NB][kTile];  // u of the blocks, twice: seldom looked at, so not in registers
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, j = lane >> 4;
    // the head's first block, its first channel there, the blocks it lies in
    const int hd = PART ? a.hd : HD, b0 = PART ? blockIdx.x * hd / 32 : blockIdx.x * NB, shift = PART ? blockIdx.x * hd % 32 : 0;
    const int nb = PART ? (shift + hd + 31) / 32 : NB;
    const int kh = blockIdx.x, row0 = blockIdx.y * kTile, rows = a.n_tokens * a.group;
    const int pos = a.d_pos ? *a.d_pos : a.pos;
    const int tile_lim = pos + (min(row0 + kTile, rows) - 1) / a.group, first_lim = pos + row0 / a.group;
    const int n_split = gridDim.z, chunk = split_chunk(a, pos, n_split);
    const int begin = blockIdx.z * chunk, end = min(begin + chunk, steps_of(a.map, tile_lim));
    if (begin >= end) return;  // rows past the tile's last position

    const int groups = a.map.groups, last_group = a.map.group_of(tile_lim);
    const size_t sc_off = kv4_scales(a.map.page_tokens, a.kv_dim);
    const size_t n_head_off = static_cast<size_t>(b0) * groups * 128, s_head_off = sc_off + static_cast<size_t>(b0) * groups * 32;
    const size_t n_blk = static_cast<size_t>(groups) * 128, s_blk = static_cast<size_t>(groups) * 32;
    const uint32_t kn_lane = (col >> 2) * 128 + (j * 4 + (col & 3)) * 8, vn_lane = j * 128 + col * 8, s_lane = j * 32;
    const uint32_t vc_lane = static_cast<uint32_t>(min(col, nb - 1)) * static_cast<uint32_t>(s_blk) + j * 32 + 16;
    uint32_t kc_lane[(NB + 3) / 4];
#pragma unroll
    for (int k = 0; k < (NB + 3) / 4; ++k)
        kc_lane[k] = static_cast<uint32_t>(min(j + 4 * k, nb - 1)) * static_cast<uint32_t>(s_blk) + (col >> 2) * 32 + 16 + (col & 3) * 4;

    // the page of group g (of 4) of step st, and the group's index there (UNI: whole steps lie in a page)
    auto locate = [&](const void* const* pt, int st, int g, const uint8_t*& base, int& at) {
        const int vg = min(4 * st + g, last_group), page = a.map.page_of(vg);
        base = static_cast<const uint8_t*>(pt[page]);
        at = vg - page * groups;
    };
    constexpr int NQ = (NB + 3) / 4;  // blocks j, j + 4 of a lane's share of the c
    uint2 kn[NB], vn[NB];
    u32x4 ks[NB], vs[NB], vc;
    uint32_t kc[NQ];  // c of the lane's two cache rows, blocks j and j + 4
    auto load_k = [&](const uint8_t* page, int st) {
        if constexpr (UNI) {
            const int g0 = 4 * st - a.map.page_of(4 * st) * groups;
            const uint8_t* words = page + n_head_off + static_cast<size_t>(g0) * 128;
            const uint8_t* sb = page + s_head_off + static_cast<size_t>(g0) * 32;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                kn[b] = ld8_at(words + b * n_blk, kn_lane);
                ks[b] = ld16_at(sb + b * s_blk, s_lane);
            }
#pragma unroll
            for (int k = 0; k < NQ; ++k) kc[k] = ld4_at(sb, kc_lane[k]);
        } else {
            const uint8_t *bn, *bs;
            int gn, gs;
            locate(a.pt_k, st, col >> 2, bn, gn);
            locate(a.pt_k, st, j, bs, gs);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                kn[b] = ld8_at(bn + n_head_off + b * n_blk + static_cast<size_t>(gn) * 128, (j * 4 + (col & 3)) * 8);
                ks[b] = ld16_at(bs + s_head_off + b * s_blk + static_cast<size_t>(gs) * 32, 0);
            }
#pragma unroll
            for (int k = 0; k < NQ; ++k)
                kc[k] = ld4_at(bn + s_head_off + min(j + 4 * k, nb - 1) * s_blk + static_cast<size_t>(gn) * 32, 16 + (col & 3) * 4);
        }
    };
    auto load_v = [&](const uint8_t* page, int st) {
        if constexpr (UNI) {
            const int g0 = 4 * st - a.map.page_of(4 * st) * groups;
            const uint8_t* words = page + n_head_off + static_cast<size_t>(g0) * 128;
            const uint8_t* sb = page + s_head_off + static_cast<size_t>(g0) * 32;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                vn[b] = ld8_at(words + b * n_blk, vn_lane);
                vs[b] = ld16_at(sb + b * s_blk, s_lane);
            }
            vc = ld16_at(sb, vc_lane);
        } else {
            const uint8_t* base;
            int g;
            locate(a.pt_v, st, j, base, g);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                vn[b] = ld8_at(base + n_head_off + b * n_blk + static_cast<size_t>(g) * 128, col * 8);
                vs[b] = ld16_at(base + s_head_off + b * s_blk + static_cast<size_t>(g) * 32, 0);
            }
            vc = ld16_at(base + s_head_off + min(col, nb - 1) * s_blk + static_cast<size_t>(g) * 32, 16);
        }
    };
    auto page_of_step = [&](const void* const* pt, int st) -> const uint8_t* {
        if constexpr (UNI) return page_at(pt, a.map.page_of(4 * st));
        else return nullptr;
    };

    int st = begin + wave;
    if (st < end) {
        load_k(page_of_step(a.pt_k, st), st);
        load_v(page_of_step(a.pt_v, st), st);
    }

    // q: lane (col, j) holds channels 8 j .. of each block of row col; scaled by a power of two
    const int r = min(row0 + col, rows - 1), lim = pos + r / a.group;
    const float* qr = a.q + static_cast<size_t>(r / a.group) * a.q_pitch + static_cast<size_t>(kh * a.group + r % a.group) * hd - shift;
    // masks and constants that the compiler is not to see: as selects and literals they take more operations
    uint32_t c_mask = col < NB ? 0xffffffffu : 0u, c_fill = col == NB ? 0x3c003c00u : 0u;  // ones: sum p
    float minus1 = -1.0f;
    Q4Ones ones;
    asm("" : "+v"(ones.c16), "+v"(ones.c256), "+v"(c_mask), "+v"(c_fill), "+v"(minus1));
    // two numbers in two fp16 each: rounded, and what the rounding left
    auto part = [&](float a, float b, uint32_t& hi, uint32_t& lo) {
        const half2v h = pk_half(a, b);
        hi = as_u32(h);
        lo = as_u32(pk_half(less(a, h.x, minus1), less(b, h.y, minus1)));
    };
    u32x4 qh[NB], ql[NB], qch = {0u, 0u, 0u, 0u}, qcl = qch;  // qc: block sums of q, one or two a lane: the operand that meets kc
    float y_scale;
    {
        float f[NB][8], top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int c = 32 * b + 8 * j;
            const bool own = !PART || (c >= shift && c < shift + hd);  // both are multiples of 8
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[b][i] = own ? qr[c + i] : 0.0f;
                top = fmaxf(top, fabsf(f[b][i]));
            }
        }
        top = rows_max(top);
        const int e = query_exponent(top);
        const float down = ldexpf(1.0f, -e);
        y_scale = ldexpf(__fdiv_rn(kLog2e, sqrt_rn(static_cast<float>(hd))), e);
        float mine[NQ];
#pragma unroll
        for (int k = 0; k < NQ; ++k) mine[k] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[b][i] *= down;
                sum += f[b][i];
            }
            sum = rows_sum(sum);
            if ((b & 3) == j) mine[b / 4] = sum;
            uint32_t h[4], l[4];  // the order of q4_unpack
            part(f[b][0], f[b][4], h[0], l[0]);
            part(f[b][1], f[b][5], h[1], l[1]);
            part(f[b][2], f[b][6], h[2], l[2]);
            part(f[b][7], f[b][3], h[3], l[3]);
            qh[b] = u32x4{h[0], h[1], h[2], h[3]};
            ql[b] = u32x4{l[0], l[1], l[2], l[3]};
        }
        uint32_t h, l;
        part(mine[0], NQ > 1 ? mine[NQ - 1] : 0.0f, h, l);
        qch[0] = h;
        qcl[0] = l;
    }

    f32x4 o[NB][2], oc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b][0] = o[b][1] = oc;
    float m = kLowest;  // of the scores before y_scale
    bool uneven = false;  // in the wave: a u that is not 1
    auto unit = [&](int b) { return uneven ? as_half2(s_unit[wave][b][col]) : both(kUnitOne); };
    uint32_t wide = 0;    // a u below 1, by block
    const uint32_t c_turn = (col & 3) == 3 ? 16 : 0;  // rows 3 and 7 are stored the other way round

    const u32x4 zero_words = {0u, 0u, 0u, 0u};
    auto step = [&](auto edge_tag) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        const bool fresh = st == begin + wave;
        const uint8_t *next_k = nullptr, *next_v = nullptr;
        const bool more = st + kWaves < end;
        if (more) {
            next_k = page_of_step(a.pt_k, st + kWaves);
            next_v = page_of_step(a.pt_v, st + kWaves);
        }
        // scores of rows 8 j + i (s0) and 8 j + 4 + i (s1): the c first, then block by block
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        f32x4 s0, s1;
        {
            u32x4 c0 = zero_words, c1 = zero_words;
            uint32_t w0 = __builtin_amdgcn_alignbit(kc[0], kc[0], c_turn);
            if constexpr (NQ == 1) {
                c0[0] = w0 & 0xffffu;
                c1[0] = w0 >> 16;
            } else {
                const uint32_t w1 = __builtin_amdgcn_alignbit(kc[NQ - 1], kc[NQ - 1], c_turn);
                c0[0] = (w0 & 0xffffu) | (w1 << 16);
                c1[0] = (w0 >> 16) | (w1 & 0xffff0000u);
            }
            s0 = mfma2(c0, qch, qcl, zero);
            s1 = mfma2(c1, qch, qcl, zero);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (PART && b >= nb) continue;
            const f32x4 c0 = mfma2(__builtin_bit_cast(u32x4, q4_unpack(kn[b].x, ones)), qh[b], ql[b], zero);
            const f32x4 c1 = mfma2(__builtin_bit_cast(u32x4, q4_unpack(kn[b].y, ones)), qh[b], ql[b], zero);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const half2v s = as_half2(ks[b][i]);
                s0[i] = fmaf(static_cast<float>(i < 3 ? s.x : s.y), c0[i], s0[i]);
                s1[i] = fmaf(static_cast<float>(i < 3 ? s.y : s.x), c1[i], s1[i]);
            }
        }
        if (more) load_k(next_k, st + kWaves);
        // rows of the step that a query row does not see: p = 0, whatever is stored there
        uint32_t seen[4], seen_c[4];
        if constexpr (EDGE) {
            const int page = a.map.page_of(4 * st + j), g = 4 * st + j - page * groups;
            const int p0 = page * a.map.page_tokens + g * 8, room = a.map.page_tokens - g * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in0 = i < room, in1 = i + 4 < room;
                const bool v0 = in0 && p0 + i <= lim, v1 = in1 && p0 + i + 4 <= lim;
                if (!v0) s0[i] = -INFINITY;
                if (!v1) s1[i] = -INFINITY;
                const uint32_t first = i < 3 ? 0xffffu : 0xffff0000u;
                seen[i] = (v0 ? first : 0u) | (v1 ? ~first : 0u);
                seen_c[i] = (in0 && p0 + i <= tile_lim ? first : 0u) | (in1 && p0 + i + 4 <= tile_lim ? ~first : 0u);
            }
        }
        float mx = s0[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(fmaxf(mx, s0[i]), s1[i]);
        mx = rows_max(mx);
        // steps that the query row sees
        auto steps = [&](int b, int i) { return EDGE ? vs[b][i] & seen[i] : vs[b][i]; };
        // one that reaches 2 with its block's u
        uint32_t big = 0;
        if (uneven) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                const half2v u = unit(b);
#pragma unroll
                for (int i = 0; i < 4; ++i) big |= reaches_2(steps(b, i), u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    if (!PART || b < nb) w |= vs[b][i];
                big |= EDGE ? w & seen[i] : w;
            }
            big &= kWideBits;
        }
        // a row that sees nothing here sees nothing later
        auto blind = [&] {
            const int page = a.map.page_of(4 * st);
            return EDGE && lim < page * a.map.page_tokens + (4 * st - page * groups) * 8;
        };
        bool small = false;  // the first step has a block with none of 2^-7 or more
        if (fresh) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                uint64_t rows_with = __ballot(((steps(b, 0) | steps(b, 1) | steps(b, 2) | steps(b, 3)) & kUsualBits) || blind());
                rows_with |= rows_with >> 32;
                rows_with |= rows_with >> 16;
                small = small || (rows_with & 0xffff) != 0xffff;
            }
        }
        const bool ahead = (mx - m) * y_scale > kSlack;
        if (small || __any(ahead || big)) {
            const float top = ahead ? mx : m, f = __builtin_amdgcn_exp2f((m - top) * y_scale);
            m = top;
            oc *= f;
            if (small || __any(big)) {
                wide = 0;
                uint32_t other = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (PART && b >= nb) continue;
                    uint32_t most = max_half(max_halves(max_halves(steps(b, 0), steps(b, 1)), max_halves(steps(b, 2), steps(b, 3))));
                    most = rows_max_bits(most);
                    const half2v was = fresh ? both(blind() ? kUnitOne : kUnitFirst) : unit(b);
                    const half2v u = reaches_2(most, was) ? both(unit_of(most)) : was;
                    s_unit[wave][b][col] = as_u32(u);
                    const float g = f * unit_f(u) * unit_inverse(was);
                    o[b][0] *= g;
                    o[b][1] *= g;
                    other |= (as_u32(u) & 0xffffu) ^ kUnitOne;
                    if (__any(below_1(u))) wide |= 1u << b;
                }
                uneven = __any(other);
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    o[b][0] *= f;
                    o[b][1] *= f;
                }
            }
        }
        const bool far = fabsf(m * y_scale) > kFar;
        if (__any(far)) {
            const float base = far ? m : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) s0[i] -= base, s1[i] -= base;
        }
        const float below = far ? kLift : fmaf(-m, y_scale, kLift);
        if (uneven) {
            float scale = y_scale;
            asm("" : "+v"(scale));  // or the weights are formed for both here, apart from the products below
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                const half2v u = unit(b);
                if (wide >> b & 1) {
                    u32x4 fh, fl;
                    const float uw = below_1(u) ? unit_f(u) : 0.0f;  // the other query rows' below
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p0 = __builtin_amdgcn_exp2f(fmaf(s0[i], scale, below)), p1 = __builtin_amdgcn_exp2f(fmaf(s1[i], scale, below));
                        uint32_t h, l;
                        times_steps(i < 3 ? p0 : p1, i < 3 ? p1 : p0, as_half2(steps(b, i)), uw, minus1, h, l);
                        fh[i] = h;
                        fl[i] = l;
                    }
                    o[b][0] = mfma2(__builtin_bit_cast(u32x4, q4_unpack(vn[b].x, ones)), fh, fl, o[b][0]);
                    o[b][1] = mfma2(__builtin_bit_cast(u32x4, q4_unpack(vn[b].y, ones)), fh, fl, o[b][1]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) vs[b][i] = below_1(u) ? 0u : as_u32(as_half2(steps(b, i)) * u);
            }
        }
        {
            half2v hi[4], lo[4];
            u32x4 ph, pl, cf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s0[i], y_scale, below)), p1 = __builtin_amdgcn_exp2f(fmaf(s1[i], y_scale, below));
                uint32_t h, l;
                part(i < 3 ? p0 : p1, i < 3 ? p1 : p0, h, l);
                ph[i] = h;
                pl[i] = l;
                hi[i] = as_half2(h);
                lo[i] = as_half2(l);
                cf[i] = ((EDGE ? vc[i] & seen_c[i] : vc[i]) & c_mask) | c_fill;
            }
            oc = mfma2(cf, ph, pl, oc);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (PART && b >= nb) continue;
                u32x4 fh, fl;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t h, l;
                    times_steps(hi[i], lo[i], as_half2(steps(b, i)), h, l);
                    fh[i] = h;
                    fl[i] = l;
                }
                o[b][0] = mfma2(__builtin_bit_cast(u32x4, q4_unpack(vn[b].x, ones)), fh, fl, o[b][0]);
                o[b][1] = mfma2(__builtin_bit_cast(u32x4, q4_unpack(vn[b].y, ones)), fh, fl, o[b][1]);
            }
        }
        if (more) load_v(next_v, st + kWaves);
    };
    // steps that every query row sees whole; none where pages end inside a group
    const int full = a.map.page_tokens & 7 ? 0 : (first_lim + 1) / 32;
    for (; st < min(end, full); st += kWaves) step(std::false_type{});
    for (; st < end; st += kWaves) step(std::true_type{});

    // the waves joined
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const float inverse = unit_inverse(unit(b));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 v = o[b][h] * inverse;
            *reinterpret_cast<float4*>(&s_o[wave][col][32 * b + 16 * h + 4 * j]) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (4 * j + i <= NB) s_c[wave][col][4 * j + i] = oc[i];
    if (lane < kTile) s_m[wave][lane] = fmaf(m, y_scale, -kLift);
    __syncthreads();
    for (int idx = threadIdx.x; idx < kTile * HD; idx += 64 * kWaves) {
        const int c = idx / HD, d = idx % HD, row = row0 + c;
        if (row >= rows) break;
        float top = s_m[0][c], sum = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_m[w][c]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][c] - top);
            sum = fmaf(f, s_o[w][c][d] + s_c[w][c][d / 32], sum);
            l = fmaf(f, s_c[w][c][NB], l);
        }
        if (!PART || (d >= shift && d < shift + hd)) write_sum(a, kh, row, d - shift, hd, n_split, sum, l, top);
    }
}

// Few query rows (token * group + head <= 4: decoding with up to four heads a kv
// head): of the kernel above's 16 columns most would be empty, while its work
// per lane stays the same.  Here the matrix pipe takes 16 products of 4 x 4 at
// once, with the query rows as their short side and 64 cache rows a step:
//   scores  16 quads of cache rows (a lane's own row) by 4 query rows, 4
//           channels at a time; q comes from one of four 16-lane groups, so
//           that a register holds four channel steps of it;
//   values  64 channels (a lane's own) by 4 query rows, one quad of cache rows
//           at a time: its p s is broadcast to the 8 channel quads of a block.
// The scores leave a lane with four cache rows of one query row, which is the
// operand that the values take.  Rows of a group go in the order of the scales
// (0 4 1 5, 2 6 7 3), as the words unpack.  65000 rows of 8 kv heads of 128, 4
// heads each: 24.0 us with the join (alone 21.6 traced, 3.9 TB/s), with the kernel
// above 26.5.  Of its wave cycles 31 % wait, with two waves per SIMD (204
// registers) that load one step ahead; VALU 48 %, matrix pipe 16 % busy.
template <int NB, bool UNI>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_q4_narrow_kernel(Q4Args a) {
    constexpr int HD = 32 * NB, NH = NB / 2, NR = 2 * NB;  // 64-channel halves; q registers (of four channel steps)
    __shared__ float s_o[kWaves][4][HD];
    __shared__ float s_c[kWaves][4][NB];
    __shared__ float s_l[kWaves][4], s_m[kWaves][4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int head = lane & 3, half32 = lane >> 5, g8 = lane >> 3, odd = (lane >> 2) & 1;  // odd: the group's second quad
    const int kh = blockIdx.x, row0 = blockIdx.y * 4, rows = a.n_tokens * a.group;
    const int pos = a.d_pos ? *a.d_pos : a.pos;
    const int tile_lim = pos + (min(row0 + 4, rows) - 1) / a.group, first_lim = pos + row0 / a.group;
    const int n_split = gridDim.z, chunk = split_chunk(a, pos, n_split);
    const int begin = blockIdx.z * chunk, end = min(begin + chunk, steps_of(a.map, tile_lim));
    if (begin >= end) return;  // rows past the tile's last position

    const int groups = a.map.groups, last_group = a.map.group_of(tile_lim);
    const size_t sc_off = kv4_scales(a.map.page_tokens, a.kv_dim);
    const size_t n_head_off = static_cast<size_t>(kh * NB) * groups * 128, s_head_off = sc_off + static_cast<size_t>(kh * NB) * groups * 32;
    const uint32_t n_blk = static_cast<uint32_t>(groups) * 128, s_blk = static_cast<uint32_t>(groups) * 32;
    const int in_group = lane & 7;
    const uint32_t k_word = (in_group < 6 ? in_group : 13 - in_group) * 4;  // the lane's row among a group's words

    uint32_t kn[NB][4], vn[NH][8];
    uint2 ks[NB], kc[NB], vs[NH][2], vc[NQuad<NB>::value];
    auto group_at = [&](const void* const* pt, int vg, int& at) -> const uint8_t* {
        const int v = min(vg, last_group), page = a.map.page_of(v);
        at = v - page * groups;
        return static_cast<const uint8_t*>(pt[page]);
    };
    auto load_k = [&](const uint8_t* page, int it) {
        const uint8_t *nb, *sb;
        uint32_t on, os;
        if constexpr (UNI) {
            const int g0 = 8 * it - a.map.page_of(8 * it) * groups;
            nb = page + n_head_off + static_cast<size_t>(g0) * 128;
            sb = page + s_head_off + static_cast<size_t>(g0) * 32;
            on = g8 * 128 + k_word;
            os = g8 * 32 + odd * 8;
        } else {
            int g;
            const uint8_t* base = group_at(a.pt_k, 8 * it + g8, g);
            nb = base + n_head_off + static_cast<size_t>(g) * 128;
            sb = base + s_head_off + static_cast<size_t>(g) * 32;
            on = k_word;
            os = odd * 8;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int kq = 0; kq < 4; ++kq) kn[b][kq] = ld4_at(nb + static_cast<size_t>(b) * n_blk, on + kq * 32);
            ks[b] = ld8_at(sb + static_cast<size_t>(b) * s_blk, os);
            kc[b] = ld8_at(sb + static_cast<size_t>(b) * s_blk, os + 16);
        }
    };
    auto load_v = [&](const uint8_t* page, int it) {
        if constexpr (UNI) {
            const int g0 = 8 * it - a.map.page_of(8 * it) * groups;
            const uint8_t* nb = page + n_head_off + static_cast<size_t>(g0) * 128;
            const uint8_t* sb = page + s_head_off + static_cast<size_t>(g0) * 32;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
#pragma unroll
                for (int g = 0; g < 8; ++g) vn[h][g] = ld4_at(nb + static_cast<size_t>(2 * h) * n_blk, half32 * n_blk + (lane & 31) * 4 + g * 128);
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    vs[h][t] = ld8_at(sb + static_cast<size_t>(2 * h) * s_blk, half32 * s_blk + (4 * t + (g8 & 3)) * 32 + odd * 8);
            }
#pragma unroll
            for (int k = 0; k < NQuad<NB>::value; ++k)
                vc[k] = ld8_at(sb, static_cast<uint32_t>(min(head + 4 * k, NB - 1)) * s_blk + g8 * 32 + 16 + odd * 8);
        } else {
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const int v = min(8 * it + g, last_group), p = a.map.page_of(v);
                const uint8_t* nb = page_at(a.pt_v, p) + n_head_off + static_cast<size_t>(v - p * groups) * 128;
#pragma unroll
                for (int h = 0; h < NH; ++h) vn[h][g] = ld4_at(nb + static_cast<size_t>(2 * h) * n_blk, half32 * n_blk + (lane & 31) * 4);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                int g;
                const uint8_t* sb = group_at(a.pt_v, 8 * it + 4 * t + (g8 & 3), g) + s_head_off;
#pragma unroll
                for (int h = 0; h < NH; ++h)
                    vs[h][t] = ld8_at(sb + static_cast<size_t>(2 * h + half32) * s_blk + static_cast<size_t>(g) * 32, odd * 8);
            }
            int g;
            const uint8_t* sb = group_at(a.pt_v, 8 * it + g8, g) + s_head_off;
#pragma unroll
            for (int k = 0; k < NQuad<NB>::value; ++k)
                vc[k] = ld8_at(sb + static_cast<size_t>(min(head + 4 * k, NB - 1)) * s_blk + static_cast<size_t>(g) * 32, 16 + odd * 8);
        }
    };
    auto page_of_it = [&](const void* const* pt, int it) -> const uint8_t* {
        if constexpr (UNI) return page_at(pt, a.map.page_of(8 * it));
        else return nullptr;
    };

    const int it_end = (end + 1) / 2;
    int it = begin / 2 + wave;
    if (it < it_end) {
        load_k(page_of_it(a.pt_k, it), it);
        load_v(page_of_it(a.pt_v, it), it);
    }

    // q: register R of the 16-lane group w holds, for row `head`, channels 8 kq .. of block R / 2, kq = 2 (R % 2) + w / 2,
    // in unpacked order the first four (w even) or the last
    const int r = min(row0 + head, rows - 1), lim = pos + r / a.group;
    const float* qr = a.q + static_cast<size_t>(r / a.group) * a.q_pitch + static_cast<size_t>(kh * a.group + r % a.group) * HD;
    float minus1 = -1.0f;
    Q4Ones ones;
    asm("" : "+v"(ones.c16), "+v"(ones.c256), "+v"(minus1));
    auto part = [&](float x, float y, uint32_t& hi, uint32_t& lo) {
        const half2v h = pk_half(x, y);
        hi = as_u32(h);
        lo = as_u32(pk_half(less(x, h.x, minus1), less(y, h.y, minus1)));
    };
    half4v qh[NR], ql[NR];
    float qs[NB], y_scale;
    {
        float f[NR][4], top = 0.0f;
        const int w = lane >> 4;
#pragma unroll
        for (int R = 0; R < NR; ++R) {
            const float* x = qr + 32 * (R / 2) + 8 * (2 * (R % 2) + (w >> 1));
            f[R][0] = x[w & 1 ? 2 : 0];
            f[R][1] = x[w & 1 ? 6 : 4];
            f[R][2] = x[w & 1 ? 7 : 1];
            f[R][3] = x[w & 1 ? 3 : 5];
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(f[R][i]));
        }
        top = rows_max(top);
        const int e = query_exponent(top);
        const float down = ldexpf(1.0f, -e);
        y_scale = ldexpf(__fdiv_rn(kLog2e, sqrt_rn(static_cast<float>(HD))), e);
#pragma unroll
        for (int b = 0; b < NB; ++b) qs[b] = 0.0f;
#pragma unroll
        for (int R = 0; R < NR; ++R) {
            u32x2 hi, lo;
            uint32_t x, y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[R][i] *= down;
                qs[R / 2] += f[R][i];
            }
            part(f[R][0], f[R][1], x, y);
            hi[0] = x, lo[0] = y;
            part(f[R][2], f[R][3], x, y);
            hi[1] = x, lo[1] = y;
            qh[R] = __builtin_bit_cast(half4v, hi);
            ql[R] = __builtin_bit_cast(half4v, lo);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) qs[b] = rows_sum(qs[b]);
    }

    f32x4 oh[NH], ol[NH], oc[NQuad<NB>::value];
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < NH; ++h) oh[h] = ol[h] = zero;
#pragma unroll
    for (int k = 0; k < NQuad<NB>::value; ++k) oc[k] = zero;
    float m = kLowest, l = 0.0f;
    half2v unit[NH];  // u, twice, of the lane's block (2 h + half32) for query row `head`
#pragma unroll
    for (int h = 0; h < NH; ++h) unit[h] = both(kUnitOne);
    bool uneven = false;  // in the wave: a u that is not 1
    uint32_t wide = 0;    // a u below 1, by pair of blocks

    auto step = [&](auto edge_tag) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        const bool more = it + kWaves < it_end, fresh = it == begin / 2 + wave;
        const uint8_t *next_k = nullptr, *next_v = nullptr;
        if (more) {
            next_k = page_of_it(a.pt_k, it + kWaves);
            next_v = page_of_it(a.pt_v, it + kWaves);
        }
        f32x4 sc = zero;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x4 c = zero;
#pragma unroll
            for (int kq = 0; kq < 4; ++kq) {
                const u32x4 w = __builtin_bit_cast(u32x4, q4_unpack(kn[b][kq], ones));
                const half4v w0 = __builtin_bit_cast(half4v, u32x2{w[0], w[1]}), w1 = __builtin_bit_cast(half4v, u32x2{w[2], w[3]});
                const int R = 2 * b + kq / 2;
                if (kq & 1) {
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w0, ql[R], c, 0, 0, 6);
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w1, ql[R], c, 0, 0, 7);
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w0, qh[R], c, 0, 0, 6);
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w1, qh[R], c, 0, 0, 7);
                } else {
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w0, ql[R], c, 0, 0, 4);
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w1, ql[R], c, 0, 0, 5);
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w0, qh[R], c, 0, 0, 4);
                    c = __builtin_amdgcn_mfma_f32_4x4x4f16(w1, qh[R], c, 0, 0, 5);
                }
            }
            const half2v sa = as_half2(ks[b].x), sb = as_half2(ks[b].y), ca = as_half2(kc[b].x), cb = as_half2(kc[b].y);
            sc[0] = fmaf(static_cast<float>(ca.x), qs[b], fmaf(static_cast<float>(sa.x), c[0], sc[0]));
            sc[1] = fmaf(static_cast<float>(ca.y), qs[b], fmaf(static_cast<float>(sa.y), c[1], sc[1]));
            sc[2] = fmaf(static_cast<float>(cb.x), qs[b], fmaf(static_cast<float>(sb.x), c[2], sc[2]));
            sc[3] = fmaf(static_cast<float>(cb.y), qs[b], fmaf(static_cast<float>(sb.y), c[3], sc[3]));
        }
        if (more) load_k(next_k, it + kWaves);
        // rows that a query row does not see: p = 0, whatever is stored there
        uint32_t seen[2][2], seen_c[2];  // of quad pairs (the value operand: rows 32 t ..), of the lane's own quad
        if constexpr (EDGE) {
            const int ia[4] = {0, 4, 1, 5}, ib[4] = {2, 6, 7, 3};
            auto place = [&](int vg, int& p0, int& room) {
                const int page = a.map.page_of(vg), g = vg - page * groups;
                p0 = page * a.map.page_tokens + g * 8;
                room = a.map.page_tokens - g * 8;
            };
            int p0, room;
            place(8 * it + g8, p0, room);
            seen_c[0] = seen_c[1] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = odd ? ib[i] : ia[i];
                if (row >= room || p0 + row > lim) sc[i] = -INFINITY;
                if (row < room && p0 + row <= tile_lim) seen_c[i / 2] |= 0xffffu << (16 * (i & 1));
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                place(8 * it + 4 * t + (g8 & 3), p0, room);
                seen[t][0] = seen[t][1] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = odd ? ib[i] : ia[i];
                    if (row < room && p0 + row <= lim) seen[t][i / 2] |= 0xffffu << (16 * (i & 1));
                }
            }
        }
        float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        mx = fmaxf(mx, dpp_mov<0x124>(mx));  // over the quads: lanes 4 and 8 on, then the 16-lane rows
        mx = fmaxf(mx, dpp_mov<0x128>(mx));
        mx = rows_max(mx);
        // steps that the query row sees
        auto steps = [&](int h, int t, int k) {
            const uint32_t s = k ? vs[h][t].y : vs[h][t].x;
            return EDGE ? s & seen[t][k] : s;
        };
        // one that reaches 2 with its block's u; the first step has a block with none of 2^-7 or more
        uint32_t big = 0;
        bool small = false;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int t = 0; t < 2; ++t) big |= reaches_2(steps(h, t, 0), unit[h]) | reaches_2(steps(h, t, 1), unit[h]);
        // a row that sees nothing here sees nothing later
        auto blind = [&] {
            const int page = a.map.page_of(8 * it);
            return EDGE && lim < page * a.map.page_tokens + (8 * it - page * groups) * 8;
        };
        if (fresh) {
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                uint64_t rows_with = __ballot(((steps(h, 0, 0) | steps(h, 0, 1) | steps(h, 1, 0) | steps(h, 1, 1)) & kUsualBits) || blind());
                rows_with |= rows_with >> 16;
                rows_with |= rows_with >> 8;
                rows_with |= rows_with >> 4;
                small = small || (rows_with & 0xf0000000full) != 0xf0000000full;
            }
        }
        const bool ahead = (mx - m) * y_scale > kSlack;
        if (small || __any(ahead || big)) {
            const float top = ahead ? mx : m, f = __builtin_amdgcn_exp2f((m - top) * y_scale);
            m = top;
            l *= f;
            float g[NH];
#pragma unroll
            for (int h = 0; h < NH; ++h) g[h] = f;
            if (small || __any(big)) {
                wide = 0;
                uint32_t other = 0;
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    uint32_t most = max_half(max_halves(max_halves(steps(h, 0, 0), steps(h, 0, 1)), max_halves(steps(h, 1, 0), steps(h, 1, 1))));
                    // over the lanes of the block and query row: 4, 8 and 16 on
                    most = max(most, static_cast<uint32_t>(dpp_mov<0x124>(static_cast<int>(most))));
                    most = max(most, static_cast<uint32_t>(dpp_mov<0x128>(static_cast<int>(most))));
                    const auto x = __builtin_amdgcn_permlane16_swap(most, most, false, false);
                    most = max(x[0], x[1]);
                    const half2v was = fresh ? both(blind() ? kUnitOne : kUnitFirst) : unit[h];
                    if (reaches_2(most, was)) unit[h] = both(unit_of(most));
                    else unit[h] = was;
                    g[h] = f * unit_f(unit[h]) * unit_inverse(was);
                    other |= (as_u32(unit[h]) & 0xffffu) ^ kUnitOne;
                    if (__any(below_1(unit[h]))) wide |= 1u << h;
                }
                uneven = __any(other);
            }
            // of query row i: the quad's lane i, in the half of the channel's block
            auto rescale = [&](auto i_tag) {
                constexpr int I = decltype(i_tag)::value;
                const float fi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), I));
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const float gi = dpp_mov<I * 0x55>(g[h]);
                    oh[h][I] *= gi;
                    ol[h][I] *= gi;
                }
#pragma unroll
                for (int k = 0; k < NQuad<NB>::value; ++k) oc[k][I] *= fi;
            };
            rescale(std::integral_constant<int, 0>{});
            rescale(std::integral_constant<int, 1>{});
            rescale(std::integral_constant<int, 2>{});
            rescale(std::integral_constant<int, 3>{});
        }
        const bool far = fabsf(m * y_scale) > kFar;
        if (__any(far)) {
            const float base = far ? m : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[i] -= base;
        }
        const float below = far ? kLift : fmaf(-m, y_scale, kLift);
        // 32 rows' p s by the codes of one pair of blocks
        auto product = [&](int h, int t, u32x2 high, u32x2 low) {
            const half4v ah = __builtin_bit_cast(half4v, high), al = __builtin_bit_cast(half4v, low);
            auto quads = [&](auto g_tag) {
                constexpr int G = decltype(g_tag)::value;
                const u32x4 w = __builtin_bit_cast(u32x4, q4_unpack(vn[h][4 * t + G], ones));
                const half4v w0 = __builtin_bit_cast(half4v, u32x2{w[0], w[1]}), w1 = __builtin_bit_cast(half4v, u32x2{w[2], w[3]});
                ol[h] = __builtin_amdgcn_mfma_f32_4x4x4f16(al, w0, ol[h], 3, 2 * G, 0);
                oh[h] = __builtin_amdgcn_mfma_f32_4x4x4f16(ah, w0, oh[h], 3, 2 * G, 0);
                ol[h] = __builtin_amdgcn_mfma_f32_4x4x4f16(al, w1, ol[h], 3, 2 * G + 1, 0);
                oh[h] = __builtin_amdgcn_mfma_f32_4x4x4f16(ah, w1, oh[h], 3, 2 * G + 1, 0);
            };
            quads(std::integral_constant<int, 0>{});
            quads(std::integral_constant<int, 1>{});
            quads(std::integral_constant<int, 2>{});
            quads(std::integral_constant<int, 3>{});
        };
        if (uneven) {
            float scale = y_scale;
            asm("" : "+v"(scale));  // or the weights are formed for both here, apart from the products below
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                if (wide >> h & 1) {
                    const float uw = below_1(unit[h]) ? unit_f(unit[h]) : 0.0f;  // the other query rows' and block's below
                    float p[2][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t w = __float_as_uint(__builtin_amdgcn_exp2f(fmaf(sc[i], scale, below)));
                        const auto x = __builtin_amdgcn_permlane32_swap(w, w, false, false);
                        p[0][i] = __uint_as_float(x[0]);
                        p[1][i] = __uint_as_float(x[1]);
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        u32x2 fh, fl;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t x, y;
                            times_steps(p[t][2 * k], p[t][2 * k + 1], as_half2(steps(h, t, k)), uw, minus1, x, y);
                            fh[k] = x;
                            fl[k] = y;
                        }
                        product(h, t, fh, fl);
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t x = steps(h, t, 0), y = steps(h, t, 1);
                    vs[h][t].x = below_1(unit[h]) ? 0u : as_u32(as_half2(x) * unit[h]);
                    vs[h][t].y = below_1(unit[h]) ? 0u : as_u32(as_half2(y) * unit[h]);
                }
            }
        }
        {
            u32x2 ph, pl;
            {
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], y_scale, below));
                l += (p[0] + p[1]) + (p[2] + p[3]);
                uint32_t x, y;
                part(p[0], p[1], x, y);
                ph[0] = x, pl[0] = y;
                part(p[2], p[3], x, y);
                ph[1] = x, pl[1] = y;
            }
#pragma unroll
            for (int k = 0; k < NQuad<NB>::value; ++k) {
                const u32x2 c = {EDGE ? vc[k].x & seen_c[0] : vc[k].x, EDGE ? vc[k].y & seen_c[1] : vc[k].y};
                oc[k] = __builtin_amdgcn_mfma_f32_4x4x4f16(__builtin_bit_cast(half4v, pl), __builtin_bit_cast(half4v, c), oc[k], 0, 0, 0);
                oc[k] = __builtin_amdgcn_mfma_f32_4x4x4f16(__builtin_bit_cast(half4v, ph), __builtin_bit_cast(half4v, c), oc[k], 0, 0, 0);
            }
            // rows 0..31 and 32..63 of the step, each in both halves of the wave
            uint32_t dh[2][2], dl[2][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const auto x = __builtin_amdgcn_permlane32_swap(ph[k], ph[k], false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(pl[k], pl[k], false, false);
                dh[0][k] = x[0], dh[1][k] = x[1];
                dl[0][k] = y[0], dl[1][k] = y[1];
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    u32x2 fh, fl;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t x, y;
                        times_steps(as_half2(dh[t][k]), as_half2(dl[t][k]), as_half2(steps(h, t, k)), x, y);
                        fh[k] = x;
                        fl[k] = y;
                    }
                    product(h, t, fh, fl);
                }
            }
        }
        if (more) load_v(next_v, it + kWaves);
    };
    // steps that every query row sees whole; none where pages end inside a group
    const int full = a.map.page_tokens & 7 ? 0 : (first_lim + 1) / 64;
    for (; it < min(it_end, full); it += kWaves) step(std::false_type{});
    for (; it < it_end; it += kWaves) step(std::true_type{});

    // the quads' sums of p and p c, then the waves joined
    auto over_quads = [&](float v) {
        v += dpp_mov<0x124>(v);
        v += dpp_mov<0x128>(v);
        return rows_sum(v);
    };
    l = over_quads(l);
    const int ch = 32 * half32 + 16 * (lane & 1) + ((lane & 31) >> 1);
    float inverse[NH][4];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        const float x = unit_inverse(unit[h]);
        inverse[h][0] = dpp_mov<0x00>(x);
        inverse[h][1] = dpp_mov<0x55>(x);
        inverse[h][2] = dpp_mov<0xaa>(x);
        inverse[h][3] = dpp_mov<0xff>(x);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < NH; ++h) s_o[wave][i][64 * h + ch] = (oh[h][i] + ol[h][i]) * inverse[h][i];
#pragma unroll
        for (int k = 0; k < NQuad<NB>::value; ++k) {
            const float v = over_quads(oc[k][i]);
            if (lane < 4 && lane + 4 * k < NB) s_c[wave][i][lane + 4 * k] = v;
        }
    }
    if (lane < 4) {
        s_m[wave][lane] = fmaf(m, y_scale, -kLift);
        s_l[wave][lane] = l;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < 4 * HD; idx += 64 * kWaves) {
        const int c = idx / HD, d = idx % HD, row = row0 + c;
        if (row >= rows) break;
        float top = s_m[0][c], sum = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_m[w][c]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][c] - top);
            sum = fmaf(f, s_o[w][c][d] + s_c[w][c][d / 32], sum);
            den = fmaf(f, s_l[w][c], den);
        }
        write_sum(a, kh, row, d, HD, n_split, sum, den, top);
    }
}

// Many query rows (a prefill chunk): 32 a workgroup, on 32 x 32 products, each
// of its eight waves over every eighth step of 32 cache rows.  Against 16 rows
// a tile the unpacking of a step, a third of its operations, serves twice the
// rows.  The products' rows are the step's cache rows in the order that leaves a
// lane (query row lane % 32, half j2) with those of groups j2 and 2 + j2 in the
// order of the scales: again the next product's operand, and one 16-byte load
// of steps or middles.  q lies in LDS for all waves; a step's scales go
// through LDS too, where 32 lanes read the same ones (from the caches such
// loads would take as long as the arithmetic).  256 tokens at 1700, 32 heads on 8
// of 128: 29.5 us (16 rows a tile: 38.5), of which 9 start and end; at 16000: 180.
// A step of 32 x 32 takes a wave 460 VALU operations beside 37 matrix
// instructions, which run in turn (VALU 44 %, matrix pipe 21 % busy at 1700, 52 and
// 31 % at 16000): 256 registers, with 21 .. 22 spilled around the loops of heads of
// 128 and none in the one of whole steps, and 147 KB of LDS leave two waves per
// SIMD and a workgroup a CU (four waves a workgroup: 1.15 times as long).
constexpr int kRows32 = 32, kWaves32 = 8;
enum class Pages { kSteps, kGroups, kRows };  // pages of whole steps, of whole groups of 8 rows, of any number of rows
template <int NB, Pages PAGES>
__global__ __launch_bounds__(64 * kWaves32, 2) void attn_q4_tile_kernel(Q4Args a) {
    constexpr bool UNI = PAGES == Pages::kSteps;
    constexpr int HD = 32 * NB, NO = 16 * NB, SCALES = NB * 128;  // bytes of a step's scales of K, or of V
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    __shared__ __align__(16) uint8_t s_mem[kWaves32 * NO * 256 + kWaves32 * 6 * 256];
    __shared__ uint32_t s_unit[kWaves32][NB][kRows32];  // u of the blocks, twice: seldom looked at, so not in registers
    static_assert(kWaves32 * NO * 256 >= NB * 4 * 1024 + kWaves32 * 2 * SCALES);
    u32x4(*s_q)[2][64] = reinterpret_cast<u32x4(*)[2][64]>(s_mem);  // [block * 2 + ks][high, low][lane]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, j2 = lane >> 5;
    uint8_t* const s_sc = s_mem + NB * 4 * 1024 + wave * 2 * SCALES;  // this wave's [K, V][block][group][s, c]
    const int kh = blockIdx.x, row0 = blockIdx.y * kRows32, rows = a.n_tokens * a.group;
    const int pos = a.d_pos ? *a.d_pos : a.pos;
    const int tile_lim = pos + (min(row0 + kRows32, rows) - 1) / a.group, first_lim = pos + row0 / a.group;
    const int n_split = gridDim.z, chunk = split_chunk(a, pos, n_split);
    const int begin = blockIdx.z * chunk, end = min(begin + chunk, steps_of(a.map, tile_lim));
    if (begin >= end) return;  // rows past the tile's last position

    const int groups = a.map.groups, last_group = a.map.group_of(tile_lim);
    const size_t sc_off = kv4_scales(a.map.page_tokens, a.kv_dim);
    const size_t n_head_off = static_cast<size_t>(kh * NB) * groups * 128, s_head_off = sc_off + static_cast<size_t>(kh * NB) * groups * 32;
    const size_t n_blk = static_cast<size_t>(groups) * 128, s_blk = static_cast<size_t>(groups) * 32;
    // the cache row that row `col` of the score product is: its group of the step, its place in the scales' order, its word
    const int kg = (col >> 4) * 2 + ((col >> 2) & 1), kr = ((col >> 3) & 1) * 4 + (col & 3);
    const uint32_t k_word = (kr < 6 ? kr : 13 - kr) * 4, v_word = kv4_v_word(col) * 4;
    const int sl_b = (lane >> 4) & (NB - 1), sl_g = (lane >> 2) & 3, sl_p = (lane & 3) * 8;  // the lane's 8 bytes of scales

    uint32_t kn[NB][2], vn[NB][2];
    uint2 ksc, vsc;
    auto group_at = [&](const void* const* pt, int vg, int& at) -> const uint8_t* {
        const int v = min(vg, last_group), page = a.map.page_of(v);
        at = v - page * groups;
        return static_cast<const uint8_t*>(pt[page]);
    };
    auto load = [&](const void* const* pt, const uint8_t* page, int st, uint32_t (&w)[NB][2], bool is_k) {
        if constexpr (UNI) {
            const int g0 = 4 * st - a.map.page_of(4 * st) * groups;
            const uint8_t* nb = page + n_head_off + static_cast<size_t>(g0) * 128;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    w[b][k] = ld4_at(nb + b * n_blk, is_k ? kg * 128 + (2 * k + j2) * 32 + k_word : (2 * k + j2) * 128 + v_word);
        } else {
            int g;
            const uint8_t* base = group_at(pt, 4 * st + (is_k ? kg : j2), g) + n_head_off;
            const uint8_t* base1 = base;
            int g1 = g;
            if (!is_k) base1 = group_at(pt, 4 * st + 2 + j2, g1) + n_head_off;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                w[b][0] = ld4_at(base + b * n_blk + static_cast<size_t>(g) * 128, is_k ? j2 * 32 + k_word : v_word);
                w[b][1] = ld4_at(base1 + b * n_blk + static_cast<size_t>(g1) * 128, is_k ? (2 + j2) * 32 + k_word : v_word);
            }
        }
    };
    auto load_scales = [&](const void* const* pt, const uint8_t* page, int st) {
        if constexpr (UNI) {
            const int g0 = 4 * st - a.map.page_of(4 * st) * groups;
            return ld8_at(page + s_head_off + static_cast<size_t>(g0) * 32, sl_b * static_cast<uint32_t>(s_blk) + sl_g * 32 + sl_p);
        } else {
            int g;
            const uint8_t* sb = group_at(pt, 4 * st + sl_g, g) + s_head_off;
            return ld8_at(sb + sl_b * s_blk + static_cast<size_t>(g) * 32, sl_p);
        }
    };
    auto page_of_step = [&](const void* const* pt, int st) -> const uint8_t* {
        if constexpr (UNI) return page_at(pt, a.map.page_of(4 * st));
        else return nullptr;
    };
    // each wave's loads run a step ahead (past its last step: the same rows again), page addresses two
    int st = begin + wave;
    auto after = [&](int s) { return s + kWaves32 < end ? s + kWaves32 : s; };
    const uint8_t *next_k = nullptr, *next_v = nullptr;
    // masks and constants that the compiler is not to see: as selects and literals they take more operations
    uint32_t c_mask = col < NB ? 0xffffffffu : 0u, c_fill = col == NB ? 0x3c003c00u : 0u;  // ones: sum p
    float minus1 = -1.0f;
    Q4Ones ones;
    asm("" : "+v"(ones.c16), "+v"(ones.c256), "+v"(c_mask), "+v"(c_fill), "+v"(minus1));
    auto part = [&](float x, float y, uint32_t& hi, uint32_t& lo) {
        const half2v h = pk_half(x, y);
        hi = as_u32(h);
        lo = as_u32(pk_half(less(x, h.x, minus1), less(y, h.y, minus1)));
    };
    // q: pieces of 16 channels, half of a block, a wave's own one (lane (col, j2): channels 8 j2 .. of row col); the row's
    // maximum and the block sums go through LDS.  Scaled by a power of two
    const int r = min(row0 + col, rows - 1), lim = pos + r / a.group;
    uint32_t qch, qcl;  // block sums of blocks j2 and j2 + 2, in two parts: the operand that meets the c of K
    float y_scale;
    {
        static_assert(2 * NB <= kWaves32);
        const float* qr = a.q + static_cast<size_t>(r / a.group) * a.q_pitch + static_cast<size_t>(kh * a.group + r % a.group) * HD;
        float(*s_top)[64] = reinterpret_cast<float(*)[64]>(s_mem + kWaves32 * NO * 256), (*s_sum)[64] = s_top + 2 * NB;
        float f[8], top = 0.0f;
        if (wave < 2 * NB) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = qr[16 * wave + 8 * j2 + i];
        }
        if (st < end) {
            const uint8_t *pk = page_of_step(a.pt_k, st), *pv = page_of_step(a.pt_v, st);
            next_k = page_of_step(a.pt_k, after(st));
            next_v = page_of_step(a.pt_v, after(st));
            ksc = load_scales(a.pt_k, pk, st);
            vsc = load_scales(a.pt_v, pv, st);
            load(a.pt_k, pk, st, kn, true);
            load(a.pt_v, pv, st, vn, false);
        }
        if (wave < 2 * NB) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
            s_top[wave][lane] = top;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k) top = fmaxf(top, fmaxf(s_top[k][col], s_top[k][col + 32]));
        const int e = query_exponent(top);
        const float down = ldexpf(1.0f, -e);
        y_scale = ldexpf(__fdiv_rn(kLog2e, sqrt_rn(static_cast<float>(HD))), e);
        if (wave < 2 * NB) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] *= down;
                sum += f[i];
            }
            s_sum[wave][lane] = sum;
            uint32_t h[4], l[4];
            part(f[0], f[4], h[0], l[0]);
            part(f[1], f[5], h[1], l[1]);
            part(f[2], f[6], h[2], l[2]);
            part(f[7], f[3], h[3], l[3]);
            s_q[wave][0][lane] = u32x4{h[0], h[1], h[2], h[3]};
            s_q[wave][1][lane] = u32x4{l[0], l[1], l[2], l[3]};
        }
        __syncthreads();
        float mine[2] = {0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < NB / 2; ++x) {
            const int k = 2 * (j2 + 2 * x);
            mine[x] = (s_sum[k][col] + s_sum[k][col + 32]) + (s_sum[k + 1][col] + s_sum[k + 1][col + 32]);
        }
        part(mine[0], mine[1], qch, qcl);
    }

    f32x16 o[NB], oc;
    const f32x16 zero = {};
    oc = zero;
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = zero;
    float m = kLowest;
    half2v most_unit = both(kUnitOne);  // of the lane's block of scales: no query row's u is larger
    bool uneven = false;  // in the wave: a u that is not 1
    auto unit = [&](int b) { return uneven ? as_half2(s_unit[wave][b][col]) : both(kUnitOne); };
    uint32_t wide = 0;    // a u below 1, by block
    auto mfma = [](u32x4 x, u32x4 y, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c, 0, 0, 0);
    };
    // steps (c == 0) or middles of the rows that the lane's scores belong to: half k of them
    auto scales = [&](int which, int b, int k, int c) {
        return *reinterpret_cast<const u32x4*>(s_sc + which * SCALES + (b * 4 + 2 * k + j2) * 32 + 16 * c);
    };

    // the rows that group vg has on its page: 1 .. 8, or more
    auto room_of = [&](int vg) { return a.map.page_tokens - (vg - a.map.page_of(vg) * groups) * 8; };
    // EDGE: rows that some query rows do not see; PAD: pages that end inside a group, whose other slots hold anything: their
    // scales are cleared on the way into LDS (pages of 20 rows, 256 tokens at 16000: 246 us; with every step an EDGE 406)
    auto step = [&](auto kind_tag) {
        constexpr bool EDGE = decltype(kind_tag)::value == 2, PAD = decltype(kind_tag)::value == 1;
        const int nst = after(st);
        u32x4 qv[2][4], ks[2][2];
        auto load_q = [&](int b, u32x4 (&v)[4], u32x4 (&s)[2]) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v[2 * k] = s_q[2 * b + k][1][lane];
                v[2 * k + 1] = s_q[2 * b + k][0][lane];
                s[k] = scales(0, b, k, 0);
            }
        };
        // this wave's own memory: its reads of the last step are done, and reads follow writes in order
        bool big_step = false;
        // of the lane's pairs of rows (0, 4), (1, 5) or (2, 6), (7, 3), those below n
        auto rows_below = [&](int n, uint32_t& x, uint32_t& y) {
            const int first = (sl_p & 8) / 4;
            x = (first < n ? 0xffffu : 0u) | (first + 4 < n ? 0xffff0000u : 0u);
            y = first ? (7 < n ? 0xffffu : 0u) | (3 < n ? 0xffff0000u : 0u) : (1 < n ? 0xffffu : 0u) | (5 < n ? 0xffff0000u : 0u);
        };
        if constexpr (PAD) {  // their steps and middles: 0
            uint32_t x, y;
            rows_below(room_of(4 * st + sl_g), x, y);
            ksc.x &= x, ksc.y &= y, vsc.x &= x, vsc.y &= y;
        }
        if (NB == 4 || lane < 32) {
            *reinterpret_cast<uint2*>(s_sc + (sl_b * 4 + sl_g) * 32 + sl_p) = ksc;
            *reinterpret_cast<uint2*>(s_sc + SCALES + (sl_b * 4 + sl_g) * 32 + sl_p) = vsc;
            big_step = sl_p < 16 && reaches_2(max_halves(vsc.x, vsc.y), most_unit);
        }
        const bool fresh = st == begin + wave;
        bool small = false;  // the first step has a block with none of 2^-7 or more in the rows that all query rows see
        if (fresh) {
            uint32_t x = 0xffffffffu, y = x;
            if constexpr (EDGE) {
                const int vg = 4 * st + sl_g, page = a.map.page_of(vg), g = vg - page * groups;
                rows_below(min(a.map.page_tokens - g * 8, first_lim + 1 - page * a.map.page_tokens - g * 8), x, y);
            }
            const uint64_t with = __ballot(sl_p < 16 && (((vsc.x & x) | (vsc.y & y)) & kUsualBits));
#pragma unroll
            for (int b = 0; b < NB; ++b) small = small || !(with >> (16 * b) & 0xffff);
        }
        __builtin_amdgcn_wave_barrier();
        const uint16_t* c = reinterpret_cast<const uint16_t*>(s_sc + (j2 * 4 + kg) * 32 + 16) + kr;
        uint32_t cw = c[0];
        if constexpr (NB == 4) cw |= static_cast<uint32_t>(c[2 * 4 * 16]) << 16;
        load_q(0, qv[0], ks[0]);
        ksc = load_scales(a.pt_k, next_k, nst);
        vsc = load_scales(a.pt_v, next_v, nst);
        asm("" : "+v"(qch), "+v"(qcl));  // or the operand's four registers are kept over the loop, and others spilled
        f32x16 sc = mfma(u32x4{cw, cw, 0u, 0u}, u32x4{qch, qcl, 0u, 0u}, zero), xs[2];
        auto add = [&](const f32x16& x, const u32x4 (&s)[2]) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const half2v h = as_half2(s[k][i]);
                    sc[8 * k + 2 * i] = fmaf(static_cast<float>(h.x), x[8 * k + 2 * i], sc[8 * k + 2 * i]);
                    sc[8 * k + 2 * i + 1] = fmaf(static_cast<float>(h.y), x[8 * k + 2 * i + 1], sc[8 * k + 2 * i + 1]);
                }
        };
        // a block's products run while the last one's are scaled and the next one's q is read
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            u32x4 sb[2] = {ks[(b + 1) & 1][0], ks[(b + 1) & 1][1]};
            if (b + 1 < NB) load_q(b + 1, qv[(b + 1) & 1], ks[(b + 1) & 1]);
            f32x16 x = zero;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u32x4 w = __builtin_bit_cast(u32x4, q4_unpack(kn[b][k], ones));
                x = mfma(w, qv[b & 1][2 * k], x);
                x = mfma(w, qv[b & 1][2 * k + 1], x);
            }
            xs[b & 1] = x;
            if (b > 0) add(xs[(b + 1) & 1], sb);
            __builtin_amdgcn_sched_barrier(0);
        }
        load(a.pt_k, next_k, nst, kn, true);
        add(xs[(NB - 1) & 1], ks[(NB - 1) & 1]);
        // rows that a query row does not see: p = 0, whatever is stored there
        uint32_t seen[2][4], seen_c[2][4];
        if constexpr (PAD) {
            const int order[8] = {0, 4, 1, 5, 2, 6, 7, 3};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int room = room_of(4 * st + 2 * k + j2);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (order[i] >= room) sc[8 * k + i] = -INFINITY;
            }
        }
        if constexpr (EDGE) {
            const int order[8] = {0, 4, 1, 5, 2, 6, 7, 3};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int vg = 4 * st + 2 * k + j2, page = a.map.page_of(vg), g = vg - page * groups;
                const int p0 = page * a.map.page_tokens + g * 8, room = a.map.page_tokens - g * 8;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    seen[k][i] = seen_c[k][i] = 0;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int row = order[2 * i + x];
                        const uint32_t bits = x ? 0xffff0000u : 0xffffu;
                        if (row < room && p0 + row <= tile_lim) seen_c[k][i] |= bits;
                        if (row < room && p0 + row <= lim) seen[k][i] |= bits;
                        else sc[8 * k + 2 * i + x] = -INFINITY;
                    }
                }
            }
        }
        float mx = sc[0];
#pragma unroll
        for (int i = 1; i < 15; i += 2) mx = fmaxf(fmaxf(mx, sc[i]), sc[i + 1]);
        mx = fmaxf(mx, sc[15]);
        {
            const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
        }
        const bool ahead = (mx - m) * y_scale > kSlack;
        if (small || __any(ahead || big_step)) {
            const float top = ahead ? mx : m, f = __builtin_amdgcn_exp2f((m - top) * y_scale);
            m = top;
            oc *= f;
            if (small || __any(big_step)) {
                half2v start = both(kUnitFirst);
                if constexpr (EDGE) {  // a row that sees nothing here sees nothing later
                    const int page = a.map.page_of(4 * st);
                    if (lim < page * a.map.page_tokens + (4 * st - page * groups) * 8) start = both(kUnitOne);
                    if (fresh) most_unit = both(kUnitFirst);
                }
                wide = 0;
                uint32_t other = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t most = 0;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const u32x4 s = scales(1, b, k, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) most = max_halves(most, EDGE ? s[i] & seen[k][i] : s[i]);
                    }
                    most = max_half(most);
                    const auto t = __builtin_amdgcn_permlane32_swap(most, most, false, false);
                    most = max(t[0], t[1]);
                    const half2v was = fresh ? start : unit(b), u = reaches_2(most, was) ? both(unit_of(most)) : was;
                    s_unit[wave][b][col] = as_u32(u);
                    o[b] *= f * unit_f(u) * unit_inverse(was);
                    other |= (as_u32(u) & 0xffffu) ^ kUnitOne;
                    if (__any(below_1(u))) wide |= 1u << b;
                    if (!EDGE && sl_b == b) most_unit = u;  // one for all query rows
                }
                uneven = __any(other);
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= f;
            }
        }
        const bool far = fabsf(m * y_scale) > kFar;
        if (__any(far)) {
            const float base = far ? m : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] -= base;
        }
        const float below = far ? kLift : fmaf(-m, y_scale, kLift);
        half2v times[NB];  // where rows differ in what they see, each query row's own; 0: formed here
#pragma unroll
        for (int b = 0; b < NB; ++b) times[b] = both(kUnitOne);
        if (uneven) {
            float scale = y_scale;
            asm("" : "+v"(scale));  // or the weights are formed for both here, apart from the products below
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!(wide >> b & 1)) continue;
                const half2v u = unit(b);
                const float uw = below_1(u) ? unit_f(u) : 0.0f;  // the other query rows' below
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x4 s = scales(1, b, k, 0);
                    u32x4 fh, fl;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t h, l;
                        times_steps(__builtin_amdgcn_exp2f(fmaf(sc[8 * k + 2 * i], scale, below)),
                                    __builtin_amdgcn_exp2f(fmaf(sc[8 * k + 2 * i + 1], scale, below)),
                                    as_half2(EDGE ? s[i] & seen[k][i] : s[i]), uw, minus1, h, l);
                        fh[i] = h;
                        fl[i] = l;
                    }
                    const u32x4 w = __builtin_bit_cast(u32x4, q4_unpack(vn[b][k], ones));
                    o[b] = mfma(w, fl, o[b]);
                    o[b] = mfma(w, fh, o[b]);
                }
            }
            if constexpr (EDGE) {
#pragma unroll
                for (int b = 0; b < NB; ++b) times[b] = as_half2(below_1(unit(b)) ? 0u : as_u32(unit(b)));
            }
            __builtin_amdgcn_wave_barrier();  // the steps above are read before other lanes change them
            if (!EDGE && sl_p < 16 && (NB == 4 || lane < 32)) {
                uint2* const s = reinterpret_cast<uint2*>(s_sc + SCALES + (sl_b * 4 + sl_g) * 32 + sl_p);
                *s = below_1(most_unit) ? make_uint2(0u, 0u)
                                        : make_uint2(as_u32(as_half2(s->x) * most_unit), as_u32(as_half2(s->y) * most_unit));
            }
            __builtin_amdgcn_wave_barrier();
        }
        {
            u32x4 ph[2], pl[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t h, l;
                    part(__builtin_amdgcn_exp2f(fmaf(sc[8 * k + 2 * i], y_scale, below)),
                         __builtin_amdgcn_exp2f(fmaf(sc[8 * k + 2 * i + 1], y_scale, below)), h, l);
                    ph[k][i] = h;
                    pl[k][i] = l;
                }
                u32x4 c = *reinterpret_cast<const u32x4*>(s_sc + SCALES + (min(col, NB - 1) * 4 + 2 * k + j2) * 32 + 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = ((EDGE ? c[i] & seen_c[k][i] : c[i]) & c_mask) | c_fill;
                oc = mfma(c, pl[k], oc);
                oc = mfma(c, ph[k], oc);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x4 s = scales(1, b, k, 0);
                    u32x4 fh, fl;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        half2v z = as_half2(s[i]);
                        if constexpr (EDGE) z = as_half2(s[i] & seen[k][i]) * times[b];
                        uint32_t h, l;
                        times_steps(as_half2(ph[k][i]), as_half2(pl[k][i]), z, h, l);
                        fh[i] = h;
                        fl[i] = l;
                    }
                    const u32x4 w = __builtin_bit_cast(u32x4, q4_unpack(vn[b][k], ones));
                    o[b] = mfma(w, fl, o[b]);
                    o[b] = mfma(w, fh, o[b]);
                }
            }
        }
        load(a.pt_v, next_v, nst, vn, false);
        next_k = page_of_step(a.pt_k, after(nst));
        next_v = page_of_step(a.pt_v, after(nst));
        __builtin_amdgcn_wave_barrier();
    };
    // steps that every query row sees whole, then the others
    const int full = min(end, a.map.group_of(first_lim + 1) / 4);
    for (; st < full; st += kWaves32) step(std::integral_constant<int, PAGES == Pages::kRows ? 1 : 0>{});
    for (; st < end; st += kWaves32) step(std::integral_constant<int, 2>{});

    // the waves joined: every wave's sums by register and lane, then each wave an eighth of the registers
    __syncthreads();
    float(*s_o)[NO][64] = reinterpret_cast<float(*)[NO][64]>(s_mem);
    float(*s_x)[6][64] = reinterpret_cast<float(*)[6][64]>(s_mem + kWaves32 * NO * 256);  // sums of p c and p (rows 0..7), m
    float inverse[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) inverse[b] = unit_inverse(unit(b));
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s_o[wave][16 * b + i][lane] = o[b][i] * inverse[b];
#pragma unroll
    for (int i = 0; i < 4; ++i) s_x[wave][i][lane] = oc[i];
    s_x[wave][4][lane] = fmaf(m, y_scale, -kLift);
    __syncthreads();
    float w[kWaves32], top = s_x[0][4][lane], l = 0.0f;
#pragma unroll
    for (int k = 1; k < kWaves32; ++k) top = fmaxf(top, s_x[k][4][lane]);
    auto extra = [&](int k, int row) { return s_x[k][row & 3][col + 32 * (row >> 2)]; };
#pragma unroll
    for (int k = 0; k < kWaves32; ++k) {
        w[k] = __builtin_amdgcn_exp2f(s_x[k][4][lane] - top);
        l = fmaf(w[k], extra(k, NB), l);
    }
    const int row = row0 + col;
    if (row >= rows) return;
    const size_t out_row = static_cast<size_t>(row / a.group) * a.n_head + kh * a.group + row % a.group;
    const size_t at = out_row * n_split + blockIdx.z;
    float* dst = a.part ? a.part + at * HD : a.out + out_row * HD;
#pragma unroll
    for (int i = 0; i < NO / kWaves32; i += 4) {
        const int reg = wave * (NO / kWaves32) + i, b = reg / 16;
        float c = 0.0f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kWaves32; ++k) {
            c = fmaf(w[k], extra(k, b), c);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = fmaf(w[k], s_o[k][reg + x][lane], v[x]);
        }
        // registers 4 q .. of a block: channels 8 q + 4 j2 ..; rows of the output are only known to be 4-byte aligned
        typedef f32x4 f32x4_at4 __attribute__((aligned(4)));
        f32x4 r;  // divided as the join does it: a row has the same bits whether its call has one split or more
#pragma unroll
        for (int x = 0; x < 4; ++x) r[x] = a.part ? v[x] + c : __fdiv_rn(v[x] + c, l);
        *reinterpret_cast<f32x4_at4*>(dst + 32 * b + 2 * (reg % 16) + 4 * j2) = r;
    }
    if (a.part && wave == 0 && j2 == 0) {
        float* ml = a.part + static_cast<size_t>(a.n_tokens) * a.n_head * n_split * HD + 2 * at;
        ml[0] = top;
        ml[1] = l;
    }
}

// Heads of more than 8 blocks: a workgroup per (head, token, split), a thread a row
// for the scores, a thread a channel for the values, 256 rows at a time.  Bound
// by the unpacking, done once a head instead of once a kv head.
constexpr int kAny = 256;
__global__ __launch_bounds__(kAny) void attn_q4_any_kernel(Q4Args a) {
    extern __shared__ float s_q[];  // [hd] q, then [hd] sums
    __shared__ float s_p[kAny];
    __shared__ float s_red[kAny / 64];
    const int tid = threadIdx.x, h = blockIdx.x, t = blockIdx.y, hd = a.hd, n_split = gridDim.z;
    const int pos = a.d_pos ? *a.d_pos : a.pos, lim = pos + t;
    const int chunk = split_chunk(a, pos, n_split);
    const int begin = blockIdx.z * chunk * 4, end = min(begin + chunk * 4, a.map.group_of(lim) + 1);  // groups
    if (begin >= end) return;
    float* s_o = s_q + hd;
    for (int d = tid; d < hd; d += kAny) {
        s_q[d] = a.q[static_cast<size_t>(t) * a.q_pitch + static_cast<size_t>(h) * hd + d];
        s_o[d] = 0.0f;
    }
    __syncthreads();
    const int e0 = h / a.group * hd;  // the head's first element of a row
    const size_t sc_off = kv4_scales(a.map.page_tokens, a.kv_dim);
    const float y_scale = __fdiv_rn(kLog2e, sqrt_rn(static_cast<float>(hd)));
    float m = -INFINITY, l = 0.0f;  // the first 256 rows hold one that the token sees
    for (int g0 = begin; g0 < end; g0 += kAny / 8) {
        const int vg = min(g0 + tid / 8, end - 1), i = tid & 7;
        const int page = a.map.page_of(vg), g = vg - page * a.map.groups;
        const bool seen = g0 + tid / 8 < end && g * 8 + i < a.map.page_tokens && page * a.map.page_tokens + g * 8 + i <= lim;
        float y = -INFINITY;
        if (seen) {
            const uint8_t* base = static_cast<const uint8_t*>(a.pt_k[page]);
            float sum = 0.0f;
            for (int d = 0; d < hd; d += 8) {
                const int b = (e0 + d) / 32, kq = (e0 + d) % 32 / 8;
                const size_t at = static_cast<size_t>(b) * a.map.groups + g;
                const uint32_t w = kv4_nat(reinterpret_cast<const uint32_t*>(base + at * 128)[kv4_k_word(i, kq)]);
                const float s = kv4_step(base + sc_off + at * 32, i), c = kv4_middle(base + sc_off + at * 32, i);
                float dot = 0.0f, qsum = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float qv = s_q[d + k];
                    dot = fmaf(qv, static_cast<float>((w >> (4 * k)) & 15u) - 8.0f, dot);
                    qsum += qv;
                }
                sum = fmaf(s, dot, fmaf(c, qsum, sum));
            }
            y = sum * y_scale;
        }
        float mx = wave_max_all(y);
        if ((tid & 63) == 0) s_red[tid >> 6] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        // a NaN score reaches the sums through p, not through the maximum
        const float top = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - top);
        const float p = seen ? __builtin_amdgcn_exp2f(y - top) : 0.0f;
        s_p[tid] = p;
        __syncthreads();
        float part = 0.0f;
        for (int k = tid & 63; k < kAny; k += 64) part += s_p[k];
        part += __shfl_xor(part, 32);
        part += __shfl_xor(part, 16);
        part += __shfl_xor(part, 8);
        part += __shfl_xor(part, 4);
        part += __shfl_xor(part, 2);
        part += __shfl_xor(part, 1);
        l = fmaf(l, f, part);
        m = top;
        const int groups = min(kAny / 8, end - g0);
        for (int d = tid; d < hd; d += kAny) {
            const int b = (e0 + d) / 32, ch = (e0 + d) % 32;
            float acc = s_o[d] * f;
            for (int k = 0; k < groups; ++k) {
                const int pg = a.map.page_of(g0 + k), gg = g0 + k - pg * a.map.groups;
                const int n = min(min(8, a.map.page_tokens - gg * 8), lim - (pg * a.map.page_tokens + gg * 8) + 1);
                const uint8_t* base = static_cast<const uint8_t*>(a.pt_v[pg]);
                const size_t at = static_cast<size_t>(b) * a.map.groups + gg;
                const uint32_t w = kv4_nat(reinterpret_cast<const uint32_t*>(base + at * 128)[kv4_v_word(ch)]);
                for (int r = 0; r < n; ++r) {
                    const float s = kv4_step(base + sc_off + at * 32, r), c = kv4_middle(base + sc_off + at * 32, r);
                    acc = fmaf(s_p[8 * k + r], fmaf(s, static_cast<float>((w >> (4 * r)) & 15u) - 8.0f, c), acc);
                }
            }
            s_o[d] = acc;
        }
        __syncthreads();
    }
    const size_t row = static_cast<size_t>(t) * a.n_head + h;
    for (int d = tid; d < hd; d += kAny) {
        if (a.part) a.part[(row * n_split + blockIdx.z) * hd + d] = s_o[d];
        else a.out[row * hd + d] = __fdiv_rn(s_o[d], l);
    }
    if (a.part && tid == 0) {
        float* ml = a.part + static_cast<size_t>(a.n_tokens) * a.n_head * n_split * hd + 2 * (row * n_split + blockIdx.z);
        ml[0] = m;
        ml[1] = l;
    }
}

// The splits of a row joined: weights 2^(m - max) once in LDS, four channels a
// thread, the splits in turn over the workgroup's groups of hd / 4 threads (as
// many for any number of splits: a row's sums have one order in every chunk).  Latency is all it spends: the first
// kAhead values of a thread are on their way before the weights are known
// (one token at 65000: 24.0 us with the kernel before it; a thread a channel and no reads ahead take 0.9 more).
constexpr int kMaxSplit = 256, kJoin = 512, kAhead = 8;
__global__ __launch_bounds__(kJoin) void attn_q4_join_kernel(Q4Args a, int n_split) {
    __shared__ float s_w[kMaxSplit];
    __shared__ float s_l;
    __shared__ f32x4 s_acc[kJoin];
    const size_t row = blockIdx.x;
    const int groups = blockDim.y, d = threadIdx.x, g = threadIdx.y, tid = g * blockDim.x + d;
    const float* o = a.part + row * n_split * a.hd;
    auto value = [&](int s) { return *reinterpret_cast<const f32x4*>(o + static_cast<size_t>(s) * a.hd + 4 * d); };
    const float2* ml = reinterpret_cast<const float2*>(a.part + static_cast<size_t>(a.n_tokens) * a.n_head * n_split * a.hd) + row * n_split;
    // Reads of splits that the row does not use, which hold nothing, go ahead too: their number takes divisions
    f32x4 v[kAhead] = {};
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (g + k * groups < n_split) v[k] = value(g + k * groups);
    float2 in[kMaxSplit / 64] = {};
    if (tid < 64) {
#pragma unroll
        for (int k = 0; k < kMaxSplit / 64; ++k)
            if (tid + 64 * k < n_split) in[k] = ml[tid + 64 * k];
    }
    const int pos = a.d_pos ? *a.d_pos : a.pos, lim = pos + static_cast<int>(row) / a.n_head;
    const int chunk = split_chunk(a, pos, n_split);
    const int used = (steps_of(a.map, lim) + chunk - 1) / chunk;
    if (tid < 64) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kMaxSplit / 64; ++k)
            if (tid + 64 * k < used) top = fmaxf(top, in[k].x);
        top = wave_max_all(top);
#pragma unroll
        for (int k = 0; k < kMaxSplit / 64; ++k) {
            const int s = tid + 64 * k;
            if (s < used) {
                const float w = __builtin_amdgcn_exp2f(in[k].x - top);
                s_w[s] = w;
                sum = fmaf(w, in[k].y, sum);
            }
        }
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x);
        if (tid == 0) s_l = sum;
    }
    __syncthreads();
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float w, f32x4 x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, x[i], acc[i]);
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (g + k * groups < used) add(s_w[g + k * groups], v[k]);
#pragma unroll 4
    for (int s = g + kAhead * groups; s < used; s += groups) add(s_w[s], value(s));
    if (groups > 1) {
        s_acc[tid] = acc;
        __syncthreads();
        for (int k = 1; g == 0 && k < groups; ++k) acc += s_acc[tid + k * blockDim.x];
    }
    if (g == 0) {
        typedef f32x4 f32x4_at4 __attribute__((aligned(4)));  // rows of the output
        f32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __fdiv_rn(acc[i], s_l);
        *reinterpret_cast<f32x4_at4*>(a.out + row * a.hd + 4 * d) = r;
    }
}

// The most blocks of 32 channels that a head lies in: it starts at any multiple of the greatest common divisor
size_t q4_cover(size_t hd) { return (hd + 32 - std::gcd(hd, size_t{32}) + 31) / 32; }
bool q4_tiles(size_t hd) { return q4_cover(hd) <= 8; }

// Which kernel takes a call.  A chunk of fixed splits is to give a token the
// bits it has in any other chunk: one kernel for all (the tiles of 32 rows, where
// they take the head).  Else, by query rows of a kv head and steps of 32 cache rows:
//   up to 4 rows, from 32 steps on, the 4 x 4 products.  8 kv heads of 128,
//     1 / 4 rows, against the tiles of 16: position 1500 9.7 / 10.6 us against
//     10.3 / 10.8, 30000 15.2 / 17.3 against 17.4 / 18.1; below, fewer of the waves
//     have a step: position 100 5.7 / 6.7 against 5.4 / 5.9;
//   the tiles of 32 rows from 16 rows and 32768 rows x steps x kv heads on (they
//     unpack a step for twice the rows, but start and end slower): position 1500,
//     64 / 256 rows 15.9 / 21.0 us against 13.5 / 23.3; 16000, 8 / 16 / 32 rows
//     15.5 / 16.3 / 17.3 against 14.8 / 17.9 / 21.7; 100, 256 / 1024 rows 11.4 /
//     12.8 against 9.2 / 14.2; 4 kv heads of 64, 16000, 16 / 32 rows 12.4 / 12.0
//     against 10.7 / 12.5.
enum class Q4Kind { kNarrow, kTile16, kTile32, kAny };
Q4Kind q4_kind(size_t hd, size_t rows, size_t steps, size_t n_head_kv, size_t chunk) {
    if (!q4_tiles(hd)) return Q4Kind::kAny;
    if (hd != 64 && hd != 128) return Q4Kind::kTile16;
    if (chunk) return Q4Kind::kTile32;
    if (rows <= 4) return steps >= 32 ? Q4Kind::kNarrow : Q4Kind::kTile16;
    return rows >= 16 && rows * steps * n_head_kv >= 32768 ? Q4Kind::kTile32 : Q4Kind::kTile16;
}
size_t q4_steps(size_t max_pos, size_t page_tokens) {
    return static_cast<size_t>(kv4_map(page_tokens).group_of(static_cast<int>(max_pos - 1)) / 4 + 1);
}

// Splits of a call: enough workgroups for two a CU, each wave at least one step, at most kMaxSplit.
size_t q4_splits(size_t max_pos, size_t n_tokens, size_t n_head, size_t n_head_kv, size_t hd, size_t page_tokens,
                 size_t chunk) {
    const size_t steps = q4_steps(max_pos, page_tokens);
    if (chunk) return (steps + chunk - 1) / chunk;
    const size_t rows = n_tokens * (n_head / n_head_kv);
    size_t tiles = n_head_kv * ((rows + kTile - 1) / kTile), room = 512;
    switch (q4_kind(hd, rows, steps, n_head_kv, chunk)) {
    case Q4Kind::kTile32:  // a workgroup a CU: more splits cost more in parts than they gain
        tiles = n_head_kv * ((rows + kRows32 - 1) / kRows32);
        room = 256;
        break;
    case Q4Kind::kAny: tiles = n_head * n_tokens; break;
    default: break;
    }
    return std::max<size_t>(1, std::min({room / tiles, (steps + 2 * kWaves - 1) / (2 * kWaves), static_cast<size_t>(kMaxSplit)}));
}

template <int NB>
void q4_launch(const Q4Args& a, dim3 grid, hipStream_t st) {
    auto launch = [&](auto uni) {
        if (a.hd == 32 * NB) attn_q4_kernel<NB, decltype(uni)::value, false><<<grid, 64 * kWaves, 0, st>>>(a);
        else attn_q4_kernel<NB, decltype(uni)::value, true><<<grid, 64 * kWaves, 0, st>>>(a);
    };
    if (a.map.page_tokens % 32 == 0) launch(std::true_type{});
    else launch(std::false_type{});
}

}  // namespace

// 512 positions a split (whole 8-row groups), more where they would be over kMaxSplit
size_t attn_q4_chunk(size_t max_pos, size_t page_tokens) {
    const size_t steps = q4_steps(max_pos, page_tokens);
    size_t chunk = 16;
    while (steps > chunk * kMaxSplit) chunk *= 2;
    return chunk;
}

size_t attn_q4_scratch(size_t max_pos, size_t n_tokens, size_t n_head, size_t n_head_kv, size_t hd, size_t page_tokens,
                       size_t chunk) {
    const size_t n = q4_splits(max_pos, n_tokens, n_head, n_head_kv, hd, page_tokens, chunk);
    return n > 1 ? n * n_tokens * n_head * (hd + 2) : 0;
}

hipError_t launch_attn_q4(const void* const* pt_k, const void* const* pt_v, const float* q, size_t q_pitch, float* part,
                          float* out, const int* d_pos, size_t pos, size_t max_pos, size_t n_tokens, size_t n_head,
                          size_t n_head_kv, size_t hd, size_t kv_dim, size_t page_tokens, size_t chunk, hipStream_t st) {
    if (!n_tokens) return hipSuccess;
    const size_t splits = q4_splits(max_pos, n_tokens, n_head, n_head_kv, hd, page_tokens, chunk);
    if (hd % 8 || hd > 1024 || kv_dim % 32 || splits > static_cast<size_t>(kMaxSplit) || (splits > 1 && !part)) return hipErrorInvalidValue;
    Q4Args a{};
    a.pt_k = pt_k;
    a.pt_v = pt_v;
    a.q = q;
    a.out = out;
    a.part = splits > 1 ? part : nullptr;
    a.d_pos = d_pos;
    a.q_pitch = q_pitch;
    a.pos = static_cast<int>(pos);
    a.n_tokens = static_cast<int>(n_tokens);
    a.n_head = static_cast<int>(n_head);
    a.group = static_cast<int>(n_head / n_head_kv);
    a.kv_dim = static_cast<int>(kv_dim);
    a.hd = static_cast<int>(hd);
    a.chunk = static_cast<int>(chunk);
    a.map = kv4_map(page_tokens);
    const unsigned z = static_cast<unsigned>(splits);
    switch (q4_kind(hd, n_tokens * a.group, q4_steps(max_pos, page_tokens), n_head_kv, chunk)) {
    case Q4Kind::kNarrow: {
        const dim3 grid(static_cast<unsigned>(n_head_kv), 1, z);
        const bool uni = page_tokens % 64 == 0;
        if (hd == 128 && uni) attn_q4_narrow_kernel<4, true><<<grid, 64 * kWaves, 0, st>>>(a);
        else if (hd == 128) attn_q4_narrow_kernel<4, false><<<grid, 64 * kWaves, 0, st>>>(a);
        else if (uni) attn_q4_narrow_kernel<2, true><<<grid, 64 * kWaves, 0, st>>>(a);
        else attn_q4_narrow_kernel<2, false><<<grid, 64 * kWaves, 0, st>>>(a);
        break;
    }
    case Q4Kind::kTile32: {
        const dim3 grid(static_cast<unsigned>(n_head_kv), static_cast<unsigned>((n_tokens * a.group + kRows32 - 1) / kRows32), z);
        auto launch = [&](auto pages) {
            constexpr Pages P = decltype(pages)::value;
            if (hd == 128) attn_q4_tile_kernel<4, P><<<grid, 64 * kWaves32, 0, st>>>(a);
            else attn_q4_tile_kernel<2, P><<<grid, 64 * kWaves32, 0, st>>>(a);
        };
        if (page_tokens % 32 == 0) launch(std::integral_constant<Pages, Pages::kSteps>{});
        else if (page_tokens % 8 == 0) launch(std::integral_constant<Pages, Pages::kGroups>{});
        else launch(std::integral_constant<Pages, Pages::kRows>{});
        break;
    }
    case Q4Kind::kTile16: {
        const dim3 grid(static_cast<unsigned>(n_head_kv), static_cast<unsigned>((n_tokens * a.group + kTile - 1) / kTile), z);
        switch (q4_cover(hd)) {
        case 1: q4_launch<1>(a, grid, st); break;
        case 2: q4_launch<2>(a, grid, st); break;
        case 3: q4_launch<3>(a, grid, st); break;
        case 4: q4_launch<4>(a, grid, st); break;
        case 5:
        case 6: q4_launch<6>(a, grid, st); break;
        default: q4_launch<8>(a, grid, st); break;
        }
        break;
    }
    case Q4Kind::kAny:
        attn_q4_any_kernel<<<dim3(static_cast<unsigned>(n_head), static_cast<unsigned>(n_tokens), z), kAny,
                             2 * hd * sizeof(float), st>>>(a);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (splits > 1) {
        const size_t n4 = hd / 4, groups = std::max(std::min<size_t>(8, kJoin / n4), (63 + n4) / n4);  // a wave at least
        attn_q4_join_kernel<<<static_cast<unsigned>(n_tokens * n_head), dim3(static_cast<unsigned>(n4), static_cast<unsigned>(groups)),
                              0, st>>>(a, static_cast<int>(splits));
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace mvh
