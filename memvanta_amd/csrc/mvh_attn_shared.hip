// mvh_attn_shared.hip -- attention of a batch of sequences that share a prefix:
// every query token sees rows 0 .. prefix_len - 1 of the prefix cache and its own
// sequence's rows prefix_len .. its position (F16 and Q8 pages).
//
//   y_t = log2(e) / sqrt(hd) * q.K_t,  out = sum_t 2^(y_t - m) V_t / sum_t 2^(y_t - m)
// over both, in parts (a range of rows each) with a running m, joined at the end.
// The prefix's parts take the query rows of all sequences as the columns of one
// product, so its pages are read once per tile of rows and not once per sequence.
//
// The products run on the fp16 matrix pipe: stored fp16 values and int8 codes
// enter exactly; q and the weights are split into two fp16 (22 bits, where one
// would leave 11); sums are fp32.  A Q8 row's scale multiplies its score, and its
// weight before that is split.
#include "mvh_kernels.hpp"

namespace mvh {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
// Weights are 2^(y - m + kLift), and m follows the maximum only when that is kSlack
// ahead: at most 2^14, and in two fp16 they keep 22 bits down to 2^-12 of the
// largest, 2^-35 of it below.
constexpr float kLift = 10.0f, kSlack = 4.0f;
// From kCoarse on the base is y itself, exactly: a rounded difference could be off by more than weights may grow.
constexpr float kCoarse = 0x1p20f;
constexpr float kLeastUnit = 0x1p-126f;
constexpr int kAhead = 256;    // rows whose addresses are formed at a time, one a thread
constexpr size_t kBatch = 128;  // sequences of a launch: their places are kernel arguments

struct SharedSeq {
    const void* const* pt_k;
    const void* const* pt_v;
    int pos, row0;  // of the first query token, and its place among the tokens
};
struct SharedArgs {
    const void* const* pt_k;  // the prefix
    const void* const* pt_v;
    const float* q;
    float* out;
    float* part;  // [row][slot][hd], then [row][slot][2]: means and (m, l); null with one part
    int prefix_len, n_tokens, n_head, group, kv_heads, kv_dim, hd, slots;
    int p_page, s_page;  // rows of a page
    uint32_t p_magic, s_magic;
    int p_tiles, p_splits, p_chunk, p_items, s_tiles, s_splits, s_chunk;
    SharedSeq seq[kBatch + 1];  // row0 of the last: n_tokens
};

// A part: rows t0 .. t1 - 1 of one cache for query rows r0 .. r0 + n - 1 (row = token
// of the call * group + head of the kv head)
struct Part {
    const void* const* pt_k;
    const void* const* pt_v;
    int page;
    uint32_t magic;
    int t0, t1, r0, n, kh, slot;
    int lim0, lim_row;  // row r sees rows up to lim0 + (r - lim_row) / group
};

// t / page size, t < 2^14: magic = ceil(2^31 / that), 0 where one page holds all
__device__ __forceinline__ int page_of(int t, uint32_t magic) { return static_cast<int>(__umulhi(2 * static_cast<uint32_t>(t), magic)); }

// The order of a row's 16-byte chunks in LDS, so that the 16 rows of a K operand,
// and the 16 rows x 32 bytes of a transposed V operand, lie in different banks
template <int CPR>
__device__ __forceinline__ int k_turn(int row) { return CPR >= 16 ? row & 15 : (row >> 1) & 7; }
template <int CPR>
__device__ __forceinline__ int v_turn(int row) { return CPR >= 16 ? (row & 7) * 2 : ((row >> 1) & 3) * 2; }

// RW waves along the query rows with RT tiles of 16 each, TW along the T rows of a step
template <int RW_, int RT_, int TW_, int T_>
struct Shape {
    static constexpr int RW = RW_, RT = RT_, TW = TW_, T = T_, ROWS = 16 * RW_ * RT_;
    static constexpr bool kShared = TW_ == 1;  // all waves take all rows of a step
    static_assert(RW_ * TW_ == 4 && T_ / TW_ % 32 == 0);
};
// Bytes of each of a workgroup's two tiles: a step's K or V, or, loaded directly, both; and two waves' results
template <int NB, class S>
constexpr size_t tile_bytes() {
    const size_t kv = static_cast<size_t>(S::T) * NB * 64 * (S::kShared ? 2 : 1), join = S::TW > 1 ? 2 * S::RT * 16 * (32 * NB + 4) * 4 : 0;
    return kv > join ? kv : join;
}

// Eight int8 as fp16: a byte plus 128, in the low bits of 1024, less 1152
__device__ __forceinline__ uint4 half_of_int8(uint2 w) {
    const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u, one = 0x64646464u;
    const half2v off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    return make_uint4(as_u32(as_half2(__builtin_amdgcn_perm(one, a, 0x04010400u)) + off),
                      as_u32(as_half2(__builtin_amdgcn_perm(one, a, 0x04030402u)) + off),
                      as_u32(as_half2(__builtin_amdgcn_perm(one, b, 0x04010400u)) + off),
                      as_u32(as_half2(__builtin_amdgcn_perm(one, b, 0x04030402u)) + off));
}
__device__ __forceinline__ bool unbounded(_Float16 h) {  // an infinity or NaN
    return (__builtin_bit_cast(uint16_t, h) & 0x7c00u) == 0x7c00u;
}

// The part of a workgroup.  A step's T rows go to LDS as fp16: of F16 pages in shapes
// whose waves share them straight from memory, into one tile while the other
// is in use; else through registers, loaded a step ahead, K to one tile and V to the
// other.  CAUSAL: rows may be seen by some of the tokens only.
template <int KT, int NB, class S, bool CAUSAL>
__device__ __forceinline__ void attend(const SharedArgs& a, const Part& p, uint8_t* tile0, uint8_t* tile1, ulonglong2* s_row, float* s_sc,
                                        float (*s_ml)[2 * S::RT][16]) {
    constexpr int RW = S::RW, RT = S::RT, TW = S::TW, T = S::T, CPR = 4 * NB, HDP = 32 * NB, ITEMS = T * CPR / 256, ND = 2 * NB;
    constexpr bool Q8 = KT == kKvQ8, DIRECT = !Q8 && S::kShared;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, j = lane >> 4;
    const int rw = wave % RW, tw = wave / RW, hd = a.hd, kh = p.kh;

    // Addresses of the part's rows, 256 ahead of those in use: s_row[row % 512], and for Q8 pages their scales in s_sc.
    // Rows behind the part are its first one again, masked.
    const uint8_t *next_k = nullptr, *next_v = nullptr;  // the pages of this thread's next row
    int next_slot = 0;
    auto pages_of = [&](int first) {
        const int t = p.t0 + first + tid, tc = t < p.t1 ? t : p.t0, pg = page_of(tc, p.magic);
        next_k = static_cast<const uint8_t*>(p.pt_k[pg]);
        next_v = static_cast<const uint8_t*>(p.pt_v[pg]);
        next_slot = tc - pg * p.page;
    };
    constexpr int EB = Q8 ? 1 : 2;  // bytes of an element
    auto rows_of_pages = [&](int first) {
        const size_t off = EB * (static_cast<size_t>(next_slot) * a.kv_dim + p.kh * hd);
        s_row[(first + tid) & (2 * kAhead - 1)] = make_ulonglong2(reinterpret_cast<uint64_t>(next_k) + off, reinterpret_cast<uint64_t>(next_v) + off);
    };
    const size_t sc_off = kv_scale_offset(p.page, a.kv_dim);
    auto scales_of_pages = [&](int first) {
        if constexpr (Q8) {
            typedef const __attribute__((address_space(1))) float* from_t;
            const size_t off = sc_off + 4 * static_cast<size_t>(next_slot);
            s_sc[(first + tid) & (2 * kAhead - 1)] = *(from_t)(reinterpret_cast<uintptr_t>(next_k) + off);
            s_sc[2 * kAhead + ((first + tid) & (2 * kAhead - 1))] = *(from_t)(reinterpret_cast<uintptr_t>(next_v) + off);
        }
    };
    pages_of(0);
    rows_of_pages(0);
    scales_of_pages(0);
    if (DIRECT && hd < HDP)  // channels behind the head: no load writes them
        for (int i = tid; i < 2 * T * CPR; i += 256) {
            *reinterpret_cast<uint4*>(tile0 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(tile1 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
    __syncthreads();

    typename std::conditional<Q8, uint2, uint4>::type kr[DIRECT ? 1 : ITEMS], vr[DIRECT ? 1 : ITEMS];
    auto load = [&](int rel, uint8_t* tile) {  // rows t0 + rel ..
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = i * 256 + tid, row = at / CPR, kc = (at % CPR) ^ k_turn<CPR>(row), vc = (at % CPR) ^ v_turn<CPR>(row);
            const ulonglong2 from = s_row[(rel + row) & (2 * kAhead - 1)];
            const auto* pk = reinterpret_cast<const uint8_t*>(from.x + EB * 8 * kc);
            const auto* pv = reinterpret_cast<const uint8_t*>(from.y + EB * 8 * vc);
            if constexpr (DIRECT) {
                typedef const __attribute__((address_space(1))) void from_t;
                typedef __attribute__((address_space(3))) void to_t;
                uint8_t* const to = tile + (i * 256 + wave * 64) * 16;
                if (kc * 8 < hd) __builtin_amdgcn_global_load_lds((from_t*)pk, (to_t*)to, 16, 0, 0);
                if (vc * 8 < hd) __builtin_amdgcn_global_load_lds((from_t*)pv, (to_t*)(to + T * HDP * 2), 16, 0, 0);
            } else if constexpr (Q8) {
                kr[i] = vr[i] = make_uint2(0u, 0u);
                if (kc * 8 < hd) kr[i] = ld_global8(pk);
                if (vc * 8 < hd) vr[i] = ld_global8(pv);
            } else {
                kr[i] = vr[i] = make_uint4(0u, 0u, 0u, 0u);
                if (kc * 8 < hd) kr[i] = ld_global16(pk);
                if (vc * 8 < hd) vr[i] = ld_global16(pv);
            }
        }
    };
    auto store = [&] {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = (i * 256 + tid) * 16;
            if constexpr (Q8) {
                *reinterpret_cast<uint4*>(tile0 + at) = half_of_int8(kr[i]);
                *reinterpret_cast<uint4*>(tile1 + at) = half_of_int8(vr[i]);
            } else {
                *reinterpret_cast<uint4*>(tile0 + at) = kr[i];
                *reinterpret_cast<uint4*>(tile1 + at) = vr[i];
            }
        }
    };
    load(0, tile0);

    // q of the wave's rows times log2(e) / sqrt(hd): lane (n, j) holds channels 8 j .. of each block of 32, in two parts
    // of q 2^-e; scores s stand for y = s 2^e, exactly
    half8 qh[RT][NB], ql[RT][NB];
    float y_scale[RT], slack[RT];
    int lim[RT];
    float minus1 = -1.0f;  // a constant that the compiler is not to see: the subtraction takes a conversion in
    asm("" : "+v"(minus1));
    auto part2 = [&](float x, float y, half2v& h, half2v& l) {
        h = pk_half(x, y);
        l = pk_half(fmaf(static_cast<float>(h.x), minus1, x), fmaf(static_cast<float>(h.y), minus1, y));
    };
    const float factor = __fdiv_rn(kLog2e, sqrt_rn(static_cast<float>(hd)));
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = p.r0 + min((rw * RT + rt) * 16 + n, p.n - 1);
        lim[rt] = CAUSAL ? p.lim0 + (r - p.lim_row) / a.group : 0;
        const float* qr = a.q + (static_cast<size_t>(r / a.group) * a.n_head + kh * a.group + r % a.group) * hd;
        float f[NB][8], top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (32 * b + 8 * j < hd) {
                x = *reinterpret_cast<const float4*>(qr + 32 * b + 8 * j);
                y = *reinterpret_cast<const float4*>(qr + 32 * b + 8 * j + 4);
            }
            const float all[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[b][i] = all[i];
                top = fmaxf(top, fabsf(all[i]));
            }
        }
        const int e = query_exponent(rows_max(top));
        const float down = ldexpf(1.0f, -e);
        y_scale[rt] = ldexpf(1.0f, e);
        slack[rt] = kSlack * down;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                half2v h, l;
                part2(f[b][i] * down * factor, f[b][i + 1] * down * factor, h, l);
                qh[rt][b][i] = h.x, qh[rt][b][i + 1] = h.y;
                ql[rt][b][i] = l.x, ql[rt][b][i + 1] = l.y;
            }
    }
    const int seen_by_all = CAUSAL ? min(p.t1, p.lim0 + (p.r0 - p.lim_row) / a.group + 1) : p.t1;

    f32x4 o[RT][ND];
    float m[RT], base_y[RT], l[RT];  // the largest s (within kSlack), what is taken off y, the sum of weights
    float unit[RT], per_unit[RT];    // Q8: sums are held in units, the power of two at the largest V scale seen, and 1 / unit
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_inff();
        base_y[rt] = l[rt] = 0.0f;
        unit[rt] = kLeastUnit, per_unit[rt] = 1.0f / kLeastUnit;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[rt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // A lane's first LDS reads; those of other blocks of channels differ in bits of the chunk, those of other rows by whole rows
    const int k_first = (n * CPR + (j ^ k_turn<CPR>(n))) * 16;
    const int v_row = 4 * j + (n >> 2), v_first = (v_row * CPR + (((n >> 1) & 1) ^ v_turn<CPR>(v_row))) * 16 + (n & 1) * 8;
    auto block = [&](const uint8_t* s_k, const uint8_t* s_v, int tg, int tb) {  // rows tg .. tg + 31, at tb of the tile
        const bool edge = tg + 32 > seen_by_all;
        f32x4 s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
        // LDS reads ahead of their use, held there: else each is waited for alone
        half8 k[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                k[b][h] = *reinterpret_cast<const half8*>(s_k + ((tb * CPR * 16 + k_first) ^ (b * 64)) + h * CPR * 256);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[b][h], part ? qh[rt][b] : ql[rt][b], s[rt][h], 0, 0, 0);
        auto value = [&](int d) {  // rows of V as columns: lane (n, j) gets channel 16 d + n of rows 4 j .. and 16 + 4 j ..
            union {
                s16x4 w[2];
                half8 h;
            } v;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                typedef __attribute__((address_space(3))) s16x4 lds_t;
                v.w[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_t*)(s_v + ((tb * CPR * 16 + v_first) ^ (d * 32)) + h * CPR * 256));
            }
            return v.h;
        };
        constexpr int DV = 4, BATCHES = ND / DV;  // V comes in batches of DV operands, one ahead
        half8 v[2][DV];
        auto fetch = [&](int i) {
#pragma unroll
            for (int d = 0; d < DV; ++d) v[i & 1][d] = value(i * DV + d);
        };
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 ks[2], vs[2];
        if constexpr (Q8)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = (tg - p.t0 + 16 * h + 4 * j) & (2 * kAhead - 1);
                ks[h] = *reinterpret_cast<const f32x4*>(s_sc + at);
                vs[h] = *reinterpret_cast<const f32x4*>(s_sc + 2 * kAhead + at);
            }
        half8 ph[RT], pl[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            auto seen = [&](int h, int i) {
                const int t = tg + 16 * h + 4 * j + i;
                return t < p.t1 && (!CAUSAL || t <= lim[rt]);
            };
            float top = -__builtin_inff(), widest = 0.0f;
            if constexpr (Q8)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[rt][h][i] *= ks[h][i];
            if (edge) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[rt][h][i] = seen(h, i) ? s[rt][h][i] : -__builtin_inff();
                        if constexpr (Q8) widest = fmaxf(widest, seen(h, i) ? vs[h][i] : 0.0f);
                    }
            } else if constexpr (Q8) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) widest = fmaxf(widest, vs[h][i]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[rt][h][i]);
            // seldom so for any row: its maximum over the lanes is formed only then
            if (__any(top > m[rt] + slack[rt] || (Q8 && widest >= 2.0f * unit[rt]))) {
                top = rows_max(top);
                if constexpr (Q8) widest = rows_max(widest);
                const bool ahead = top > m[rt] + slack[rt], wider = Q8 && widest >= 2.0f * unit[rt];
                float down = 1.0f;
                if (ahead) {
                    const float y = top * y_scale[rt], next = fabsf(y) < kCoarse ? y - kLift : y;
                    down = m[rt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(base_y[rt] - next);
                    m[rt] = top;
                    base_y[rt] = next;
                }
                l[rt] *= down;
                if (wider) {  // the exponent of the widest, of an infinity's the largest there is
                    const float next = __uint_as_float(min(__float_as_uint(widest) & 0x7f800000u, 0x7e800000u));
                    down *= unit[rt] / next;
                    unit[rt] = next;
                    per_unit[rt] = 1.0f / next;
                }
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rt][d][i] *= down;
            }
            float w[8], more = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(s[rt][i >> 2][i & 3], y_scale[rt], -base_y[rt]));
                more += w[i];
            }
            l[rt] += more;
            if constexpr (Q8)
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = !edge || seen(i >> 2, i & 3) ? w[i] * (vs[i >> 2][i & 3] * per_unit[rt]) : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                half2v h, l2;
                part2(w[i], w[i + 1], h, l2);
                ph[rt][i] = h.x, ph[rt][i + 1] = h.y;
                pl[rt][i] = l2.x, pl[rt][i + 1] = l2.y;
            }
        }
        bool odd = false;
#pragma unroll
        for (int i = 0; i < BATCHES; ++i) {
            if (i + 1 < BATCHES) fetch(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (CAUSAL && !Q8 && edge) {
                // a row that some do not see: what is no number there must not meet their weight of 0
#pragma unroll
                for (int d = 0; d < DV; ++d)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (unbounded(v[i & 1][d][e])) {
                            odd = true;
                            v[i & 1][d][e] = static_cast<_Float16>(0.0f);
                        }
            }
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int d = 0; d < DV; ++d)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        o[rt][i * DV + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i & 1][d], part ? ph[rt] : pl[rt], o[rt][i * DV + d], 0, 0, 0);
        }
        if (CAUSAL && !Q8 && __any(odd)) {  // the products left out, for the rows that see them
#pragma unroll 1
            for (int t = 0; t < 32; ++t) {
                const int row = tb + t, from_lane = n + 16 * ((t >> 2) & 3), at = 4 * (t >> 4) + (t & 3);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float w = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i == at) w = static_cast<float>(ph[rt][i]) + static_cast<float>(pl[rt][i]);
                    w = __shfl(w, from_lane);
                    if (tg + t >= p.t1 || tg + t > lim[rt]) continue;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int ch = 16 * d + 4 * j + i;
                            const _Float16 x = *reinterpret_cast<const _Float16*>(
                                s_v + (row * CPR + ((ch >> 3) ^ v_turn<CPR>(row))) * 16 + (ch & 7) * 2);
                            if (unbounded(x)) o[rt][d][i] = fmaf(w, static_cast<float>(x), o[rt][d][i]);
                        }
                }
            }
        }
    };

    const int count = p.t1 - p.t0;
    // the next 256 rows: their pages in a turn of 256 rows' first step, addresses at its end, scales in the second step
    auto look_ahead = [&](int rel) {
        if (rel % kAhead == 0 && rel + kAhead < count) pages_of(rel + kAhead);
    };
    auto note_ahead = [&](int rel) {
        const int first = rel - rel % kAhead + kAhead;
        if (first >= count) return;
        if (rel % kAhead == 0) rows_of_pages(first);
        if (rel % kAhead == T) scales_of_pages(first);
    };
    if constexpr (DIRECT) {
        auto step = [&](int rel, const uint8_t* tile, uint8_t* other) {
            arrive();  // this tile's rows are there, and nobody reads the other any more
            if (rel + T < count) load(rel + T, other);
            look_ahead(rel);
#pragma unroll 1
            for (int u = 0; u < T / 32; ++u)
                if (rel + 32 * u < count) block(tile, tile + T * HDP * 2, p.t0 + rel + 32 * u, 32 * u);
            note_ahead(rel);
        };
        for (int rel = 0; rel < count; rel += 2 * T) {
            step(rel, tile0, tile1);
            if (rel + T < count) step(rel + T, tile1, tile0);
        }
        arrive();  // no load into LDS outlives the workgroup
    } else {
        for (int rel = 0; rel < count; rel += T) {
            __syncthreads();
            store();
            __syncthreads();
            if (rel + T < count) load(rel + T, tile0);
            look_ahead(rel);
#pragma unroll 1
            for (int u = 0; u < T / TW / 32; ++u) {
                const int tb = tw * (T / TW) + 32 * u;
                if (rel + tb < count) block(tile0, tile1, p.t0 + rel + tb, tb);
            }
            note_ahead(rel);
        }
    }

    // the result: of the wave, or of the TW waves that shared the rows; means, so that values near fp32's end stay in it
    const size_t gs = static_cast<size_t>(a.n_tokens) * a.n_head;
    auto put = [&](int row, int d, f32x4 mean, float top, float sum) {
        const int r = p.r0 + row;
        const size_t g = static_cast<size_t>(r / a.group) * a.n_head + kh * a.group + r % a.group;
        if (!a.part) {
            *reinterpret_cast<f32x4*>(a.out + g * hd + d) = mean;
            return;
        }
        const size_t at = g * a.slots + p.slot;
        *reinterpret_cast<f32x4*>(a.part + at * hd + d) = mean;
        if (d == 0) {
            float* ml = a.part + gs * a.slots * hd + 2 * at;
            ml[0] = top;
            ml[1] = sum;
        }
    };
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = rows_sum(l[rt]);
        if (m[rt] == -__builtin_inff()) base_y[rt] = m[rt];  // nothing seen
        const float per_sum = l[rt] == 0.0f ? 0.0f : __fdiv_rn(1.0f, l[rt]);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[rt][d][i] *= per_sum;
                if constexpr (Q8) o[rt][d][i] *= unit[rt];
            }
    }
    if constexpr (TW == 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int row = (rw * RT + rt) * 16 + n;
            if (row >= p.n) continue;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (16 * d + 4 * j < hd) put(row, 16 * d + 4 * j, o[rt][d], base_y[rt], l[rt]);
        }
    } else {
        auto means = [&](int w, int rt, int row) {  // [rt][16][HDP + 4] of wave w, two waves a tile
            return reinterpret_cast<float*>(w < 2 ? tile0 : tile1) + (((w & 1) * RT + rt) * 16 + row) * (HDP + 4);
        };
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(means(wave, rt, n) + 16 * d + 4 * j) = o[rt][d];
            if (j == 0) {
                s_ml[wave][rt][n] = base_y[rt];
                s_ml[wave][RT + rt][n] = l[rt];
            }
        }
        __syncthreads();
        for (int e = tid; e < S::ROWS * (HDP / 4); e += 256) {
            const int row = e / (HDP / 4), d = e % (HDP / 4) * 4, w0 = row / (16 * RT), rt = row / 16 % RT, c = row % 16;
            if (row >= p.n || d >= hd) continue;
            float top = s_ml[w0][rt][c];
#pragma unroll
            for (int k = 1; k < TW; ++k) top = fmaxf(top, s_ml[w0 + k * RW][rt][c]);
            float weight[TW], sum = 0.0f;
#pragma unroll
            for (int k = 0; k < TW; ++k) {
                const int w = w0 + k * RW;
                const float mine = s_ml[w][rt][c], own = s_ml[w][RT + rt][c];
                weight[k] = own == 0.0f ? 0.0f : own * (mine == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mine - top));
                sum += weight[k];
            }
            const float per_sum = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < TW; ++k) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(means(w0 + k * RW, rt, c) + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = fmaf(weight[k] * per_sum, x[i], v[i]);
            }
            put(row, d, v, top, sum);
        }
    }
}

// A workgroup: a part of the prefix for a tile of all query rows, or, behind those,
// a part of one sequence's own rows.
//
// 32 heads on 8 of 128, 64 sequences behind 8000 rows: 46 us, 127 MB at 2.8 TB/s; 12
// chunks of up to 75 tokens behind 3001: 62 us, 650 TFLOP/s of products (q and weights in
// two parts, so twice the attention's own), the matrix pipe busy 27 %, VALU 33 %: 256
// registers leave two waves a SIMD, whose products and weights overlap in part.  32 Q8
// sequences of 32 heads behind 12000: 49 us, 139 MB at 2.8 TB/s, VALU 42 % (int8 to
// fp16).  5 to 6 us of each are a workgroup's way from its pages to its first rows.
// The Q8 shapes of 128 query rows spill at heads of 65 to 128: 12 registers, in chunks 27,
// to 52 and 56 bytes of scratch.  With the join, 64 Q8 sequences behind 8000 rows take 55
// us, 49 of F16; the 12 chunks 77, 62 of F16.
template <int KT, int NB, class P, class S>
__global__ __launch_bounds__(256, NB > 4 ? 1 : 2) void attn_shared_kernel(SharedArgs a) {
    constexpr size_t kP = tile_bytes<NB, P>(), kS = tile_bytes<NB, S>();
    __shared__ __align__(16) uint8_t tile0[kP > kS ? kP : kS], tile1[kP > kS ? kP : kS];
    __shared__ ulonglong2 s_row[2 * kAhead];
    __shared__ __align__(16) float s_sc[KT == kKvQ8 ? 4 * kAhead : 4];
    __shared__ float s_ml[4 * 2 * (P::RT > S::RT ? P::RT : S::RT) * 16];
    const int item = blockIdx.x;
    Part p;
    if (item < a.p_items) {
        // the tiles of a range of rows on one XCD (workgroups go to the eight in turn), whose L2 then holds it for all of them
        const int pair = item / (8 * a.p_tiles) * 8 + item % 8, tile_at = item / 8 % a.p_tiles;
        if (pair >= a.kv_heads * a.p_splits) return;
        p.kh = pair % a.kv_heads;
        p.slot = pair / a.kv_heads;
        p.pt_k = a.pt_k, p.pt_v = a.pt_v, p.page = a.p_page, p.magic = a.p_magic;
        p.t0 = p.slot * a.p_chunk;
        p.t1 = min(p.t0 + a.p_chunk, a.prefix_len);
        p.r0 = tile_at * P::ROWS;
        p.n = min(P::ROWS, a.n_tokens * a.group - p.r0);
        p.lim0 = p.lim_row = 0;
        attend<KT, NB, P, false>(a, p, tile0, tile1, s_row, s_sc, reinterpret_cast<float(*)[2 * P::RT][16]>(s_ml));
        return;
    }
    int at = item - a.p_items;
    p.kh = at % a.kv_heads;
    at /= a.kv_heads;
    const int tile_at = at % a.s_tiles;
    at /= a.s_tiles;
    const int split = at % a.s_splits, i = at / a.s_splits;
    const int rows = (a.seq[i + 1].row0 - a.seq[i].row0) * a.group, first = tile_at * S::ROWS;
    if (first >= rows) return;
    p.slot = a.p_splits + split;
    p.pt_k = a.seq[i].pt_k, p.pt_v = a.seq[i].pt_v, p.page = a.s_page, p.magic = a.s_magic;
    p.lim0 = a.seq[i].pos, p.lim_row = a.seq[i].row0 * a.group;
    p.r0 = p.lim_row + first;
    p.n = min(S::ROWS, rows - first);
    p.t0 = a.prefix_len + split * a.s_chunk;
    p.t1 = min(p.t0 + a.s_chunk, p.lim0 + (first + p.n - 1) / a.group + 1);
    if (p.t0 >= p.t1) {  // behind the last row that is seen: a part of no weight
        for (int r = threadIdx.x; r < p.n; r += 256) {
            const size_t g = static_cast<size_t>((p.r0 + r) / a.group) * a.n_head + p.kh * a.group + (p.r0 + r) % a.group;
            float* ml = a.part + static_cast<size_t>(a.n_tokens) * a.n_head * a.slots * a.hd + 2 * (g * a.slots + p.slot);
            ml[0] = -__builtin_inff();
            ml[1] = 0.0f;
        }
        return;
    }
    attend<KT, NB, S, true>(a, p, tile0, tile1, s_row, s_sc, reinterpret_cast<float(*)[2 * S::RT][16]>(s_ml));
}

// out row = the mean of its parts' means, by their sums of weights.  `per` = hd / 4
// threads hold a row's channels, four each; `ways` such groups share the parts of a row,
// and 256 / per / ways rows (at most kJoined) a workgroup.  The parts' weights come first, 32 threads a row: formed
// by every thread for itself, 16 sequences behind 4000 rows took 27.7 us, not 25.1.  A
// part without a seen row (l = 0) has no mean.  64 sequences of 32 heads of 128 in 17
// parts: 5 us, most of it the parts' 18 MB.
constexpr int kSlots = 256, kJoined = 8;  // parts of a row, rows of a workgroup
__global__ __launch_bounds__(256) void attn_shared_join(const float* __restrict__ part, float* __restrict__ out, int rows,
                                                        int slots, int hd, int per, int per_magic, int way_bits, int many) {
    __shared__ float2 s_wl[kSlots * kJoined];  // shares of the whole, and the parts' own sums
    __shared__ f32x4 s_v[256];
    const int ways = 1 << way_bits, group = threadIdx.x * per_magic >> 16, d = (threadIdx.x - group * per) * 4;
    const int in = group >> way_bits, way = group & (ways - 1);
    const int row0 = blockIdx.x * many, here = min(many, rows - row0);
    {
        const int row = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const float2* ml = reinterpret_cast<const float2*>(part + static_cast<size_t>(rows) * slots * hd) + (static_cast<size_t>(row0) + row) * slots;
        float2* const mine = s_wl + row * slots;
        float top = -__builtin_inff(), sum = 0.0f;
        if (row < here)
            for (int k = lane; k < slots; k += 32) {
                mine[k] = ml[k];
                top = fmaxf(top, mine[k].x);
            }
        top = group_max<32>(top);
        if (row < here)
            for (int k = lane; k < slots; k += 32) {
                const float w = mine[k].x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mine[k].x - top);
                mine[k].x = mine[k].y != 0.0f ? w * mine[k].y : 0.0f;
                sum += mine[k].x;
            }
        const float per_sum = __fdiv_rn(1.0f, group_sum<32>(sum));
        if (row < here)
            for (int k = lane; k < slots; k += 32) mine[k].x *= per_sum;
    }
    __syncthreads();
    const bool on = in < here;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (on) {
        const float2* mine = s_wl + in * slots;
        const float* x = part + static_cast<size_t>(row0 + in) * slots * hd + d;
        for (int k = way; k < slots; k += 4 * ways) {
            f32x4 a[4];
            float f[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int at = k + u * ways;
                const float2 wl = mine[min(at, slots - 1)];
                const bool some = at < slots && wl.y != 0.0f;
                f[u] = some ? wl.x : 0.0f;
                a[u] = some ? *reinterpret_cast<const f32x4*>(x + static_cast<size_t>(at) * hd) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = fmaf(f[u], a[u][i], v[i]);
        }
    }
    if (ways > 1) {
        s_v[threadIdx.x] = v;
        __syncthreads();
        if (!on || way) return;
        for (int w = 1; w < ways; ++w) v += s_v[threadIdx.x + w * per];
    }
    if (!on) return;
    *reinterpret_cast<f32x4*>(out + static_cast<size_t>(row0 + in) * hd + d) = v;
}

uint32_t magic_of(size_t page_tokens) {
    return page_tokens >= 16384 || !page_tokens ? 0 : static_cast<uint32_t>(((uint64_t{1} << 31) + page_tokens - 1) / page_tokens);
}

// How a launch is cut.  A CU holds two workgroups.  Tokens one by one: the prefix in
// about a workgroup a CU, whose parts beside them are the sequences' own rows (64
// sequences behind 8000 rows: 50 us, with two a CU 65, their parts' sums to be
// joined being twice as many).  Chunks, which have few own rows: at most two a CU.
struct Cut {
    bool chunks;  // own rows in tiles of many query rows
    int p_shape;  // 0, 1, 2: tiles of up to 16, 32, more query rows
    size_t p_tiles, p_splits, p_chunk, s_tiles, s_splits, s_chunk;
    size_t slots() const { return p_splits + s_splits; }
};
constexpr int kCus = 256;
constexpr int kWide = 4;  // blocks of 32 channels up to which a wave takes two tiles of query rows
size_t rows_of(int shape, int nb) { return shape == 0 && nb <= kWide ? 16 : shape <= 1 ? 32 : nb <= kWide ? 128 : 64; }
int blocks_of(size_t hd) { return hd <= 64 ? 2 : hd <= 128 ? 4 : 8; }

Cut cut_of(const SharedCall& c) {
    Cut k{};
    const int nb = blocks_of(c.head_dim);
    const size_t group = c.n_head / c.n_head_kv;
    size_t most = 0, own = 0, tokens = 0;
    for (size_t i = 0; i < c.n_seq; ++i) {
        if (!c.n_tokens[i]) continue;
        tokens += c.n_tokens[i];
        most = std::max(most, c.n_tokens[i] * group);
        own = std::max(own, c.pos[i] + c.n_tokens[i] - c.prefix_len);
    }
    const size_t rows = tokens * group;
    k.chunks = most > 32;
    k.p_shape = k.chunks || rows > 32 ? 2 : rows > 16 ? 1 : 0;
    // parts of whole 128 rows
    auto split = [](size_t len, size_t most, size_t& splits, size_t& chunk) {
        if (!len) return void(splits = chunk = 0);
        splits = std::min((len + 127) / 128, std::max<size_t>(most, 1));
        chunk = ((len + splits - 1) / splits + 127) / 128 * 128;
        splits = (len + chunk - 1) / chunk;
    };
    const size_t p_rows = rows_of(k.p_shape, nb), s_rows = rows_of(k.chunks ? 2 : 0, nb);
    k.p_tiles = (rows + p_rows - 1) / p_rows;
    k.s_tiles = (most + s_rows - 1) / s_rows;
    const size_t p_others = k.p_tiles * c.n_head_kv;
    const size_t s_others = c.n_seq * c.n_head_kv * k.s_tiles;
    split(c.prefix_len, k.chunks ? 2 * kCus / p_others : (kCus + p_others - 1) / p_others, k.p_splits, k.p_chunk);
    split(own, (2 * kCus + s_others - 1) / s_others, k.s_splits, k.s_chunk);
    return k;
}

template <int KT, int NB>
hipError_t run_shapes(const Cut& k, const SharedArgs& a, unsigned grid, hipStream_t st) {
    constexpr bool W = NB <= kWide;
    using A = typename std::conditional<W, Shape<1, 1, 4, 128>, Shape<2, 1, 2, 64>>::type;
    using B = Shape<2, 1, 2, 64>;
    using C = typename std::conditional<W, Shape<4, 2, 1, 64>, Shape<4, 1, 1, 64>>::type;
    if (k.chunks) attn_shared_kernel<KT, NB, C, C><<<grid, 256, 0, st>>>(a);
    else if (k.p_shape == 2) attn_shared_kernel<KT, NB, C, A><<<grid, 256, 0, st>>>(a);
    else if (k.p_shape == 1) attn_shared_kernel<KT, NB, B, A><<<grid, 256, 0, st>>>(a);
    else attn_shared_kernel<KT, NB, A, A><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}
template <int KT>
hipError_t run_type(int nb, const Cut& k, const SharedArgs& a, unsigned grid, hipStream_t st) {
    return nb == 2 ? run_shapes<KT, 2>(k, a, grid, st) : nb == 4 ? run_shapes<KT, 4>(k, a, grid, st) : run_shapes<KT, 8>(k, a, grid, st);
}

// Sequences first .. first + n - 1 as a call of their own
SharedCall some(const SharedCall& c, size_t first, size_t n) {
    SharedCall s = c;
    s.seq += first, s.pos += first, s.n_tokens += first;
    s.n_seq = n;
    for (size_t i = 0; i < first; ++i) {
        s.q += c.n_tokens[i] * c.n_head * c.head_dim;
        s.out += c.n_tokens[i] * c.n_head * c.head_dim;
    }
    return s;
}
size_t tokens_of(const SharedCall& c) {
    size_t n = 0;
    for (size_t i = 0; i < c.n_seq; ++i) n += c.n_tokens[i];
    return n;
}
// Workgroups of the prefix's parts, whose tiles come in eights, and of the sequences' own
size_t prefix_items(const SharedCall& c, const Cut& k) { return (k.p_splits * c.n_head_kv + 7) / 8 * 8 * k.p_tiles; }
size_t own_items(const SharedCall& c, const Cut& k) { return c.n_seq * c.n_head_kv * k.s_tiles * k.s_splits; }

// The sequences from `first` on that go in one launch: as many as its arguments hold,
// halved until it has fewer than 2^32 threads (every sequence has the tiles of the
// longest chunk, of every kv head).  One alone has fewer than 2^20 workgroups.
SharedCall launch_of(const SharedCall& c, size_t first) {
    for (size_t n = std::min(kBatch, c.n_seq - first);; n /= 2) {
        const SharedCall s = some(c, first, n);
        const Cut k = cut_of(s);
        if (n == 1 || prefix_items(s, k) + own_items(s, k) < size_t{1} << 24) return s;
    }
}

}  // namespace

size_t attn_shared_scratch(const SharedCall& c) {
    size_t most = 0;
    for (size_t at = 0, n; at < c.n_seq; at += n) {
        const SharedCall s = launch_of(c, at);
        n = s.n_seq;
        const Cut k = cut_of(s);
        if (k.slots() > 1) most = std::max(most, tokens_of(s) * c.n_head * k.slots() * (c.head_dim + 2) * 4);
    }
    return most;
}

hipError_t launch_attn_shared(const SharedCall& call, void* scratch, hipStream_t st) {
    for (size_t first = 0, n; first < call.n_seq; first += n) {
        const SharedCall c = launch_of(call, first);
        n = c.n_seq;
        const size_t tokens = tokens_of(c);
        if (!tokens) continue;
        const Cut k = cut_of(c);
        SharedArgs a{};
        a.pt_k = c.prefix_k, a.pt_v = c.prefix_v, a.q = c.q, a.out = c.out;
        a.part = k.slots() > 1 ? static_cast<float*>(scratch) : nullptr;
        a.prefix_len = static_cast<int>(c.prefix_len), a.n_tokens = static_cast<int>(tokens);
        a.n_head = static_cast<int>(c.n_head), a.kv_heads = static_cast<int>(c.n_head_kv), a.group = a.n_head / a.kv_heads;
        a.kv_dim = static_cast<int>(c.kv_dim), a.hd = static_cast<int>(c.head_dim), a.slots = static_cast<int>(k.slots());
        a.p_page = static_cast<int>(c.p_page), a.s_page = static_cast<int>(c.s_page);
        a.p_magic = magic_of(c.p_page), a.s_magic = magic_of(c.s_page);
        a.p_tiles = static_cast<int>(k.p_tiles), a.p_splits = static_cast<int>(k.p_splits), a.p_chunk = static_cast<int>(k.p_chunk);
        a.s_tiles = static_cast<int>(k.s_tiles), a.s_splits = static_cast<int>(k.s_splits), a.s_chunk = static_cast<int>(k.s_chunk);
        a.p_items = static_cast<int>(prefix_items(c, k));
        int row = 0;
        for (size_t i = 0; i < c.n_seq; ++i) {
            a.seq[i] = {c.seq[i].pt_k, c.seq[i].pt_v, static_cast<int>(c.pos[i]), row};
            row += static_cast<int>(c.n_tokens[i]);
        }
        a.seq[c.n_seq].row0 = row;
        const size_t grid = a.p_items + own_items(c, k);
        const int nb = blocks_of(c.head_dim);
        const hipError_t e = c.kv_type == kKvQ8 ? run_type<kKvQ8>(nb, k, a, static_cast<unsigned>(grid), st)
                                                : run_type<kKvF16>(nb, k, a, static_cast<unsigned>(grid), st);
        if (e != hipSuccess) return e;
        if (a.part) {
            // the groups share a row's parts while each has two or more, and are at most kJoined rows
            const int rows = static_cast<int>(tokens * c.n_head), per = a.hd / 4, groups = 256 / per;
            int bits = 0;  // of the ways
            while (2 << bits <= groups && ((4 << bits) <= a.slots || groups >> bits > kJoined)) ++bits;
            const int many = groups >> bits;
            // thread / per, thread < 256: by 65536 / per, rounded up
            attn_shared_join<<<dim3(static_cast<unsigned>((rows + many - 1) / many)), 256, 0, st>>>(a.part, c.out, rows, a.slots, a.hd, per,
                                                                                                    (65535 + per) / per, bits, many);
            if (const hipError_t j = hipGetLastError(); j != hipSuccess) return j;
        }
    }
    return hipSuccess;
}

}  // namespace mvh
