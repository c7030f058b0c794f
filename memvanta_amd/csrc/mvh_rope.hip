// mvh_rope.hip -- rotary positions, and appending K and V to the paged cache
// with the rotation on the way (F32, F16, Q8 and Q4 pages); the stored rows
// read back as fp32.
//
// All of it moves bytes: a few operations per element.  A token's rot/2 turns
// cost ~35 double operations each, so a workgroup forms them once in LDS for
// all of its heads, while its first loads are on their way.
#include "mvh_kernels.hpp"
#include "mvh_kv4.hpp"
#include "mvh_rope.hpp"

namespace mvh {
namespace {

constexpr int kNoPages = -1;

struct RotArgs {
    RopeView rope;
    const float* q;
    float* q_out;
    const float* k;
    const float* v;
    size_t q_pitch, out_pitch, k_pitch, v_pitch;
    const int* positions;  // per token, or null: pos + token
    int pos, n_tokens, n_head, n_kv;
    void* const* pt_k;
    void* const* pt_v;
    int page_tokens, kv_dim;
};

__device__ __forceinline__ int token_pos(const RotArgs& a, int t) { return a.positions ? a.positions[t] : a.pos + t; }

// The turns of tokens t0 .. t0 + n - 1 into cs[n][rot / 2].
__device__ __forceinline__ void fill_turns(const RotArgs& a, int t0, int n, float2* cs) {
    const int half = a.rope.rot / 2;
    for (int i = threadIdx.x; i < n * half; i += blockDim.x) cs[i] = rope_turn(a.rope, token_pos(a, t0 + i / half), i % half);
}

template <int V>
struct Vec {
    float f[V];
};
template <int V>
__device__ __forceinline__ Vec<V> ld_vec(const float* p) {
    Vec<V> r;
    if constexpr (V == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        r.f[0] = a.x, r.f[1] = a.y, r.f[2] = a.z, r.f[3] = a.w;
    } else {
        r.f[0] = *p;
    }
    return r;
}
template <int V>
__device__ __forceinline__ void st_vec(float* p, const Vec<V>& r) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(r.f[0], r.f[1], r.f[2], r.f[3]);
    else *p = r.f[0];
}
template <int V>
__device__ __forceinline__ void st_half(uint16_t* p, const Vec<V>& r) {  // the F16 cache's rounding
    if constexpr (V == 4) {
        const uint32_t lo = f2h_ref(r.f[0]) | (static_cast<uint32_t>(f2h_ref(r.f[1])) << 16);
        const uint32_t hi = f2h_ref(r.f[2]) | (static_cast<uint32_t>(f2h_ref(r.f[3])) << 16);
        *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
    } else {
        *p = f2h_ref(r.f[0]);
    }
}

// Units of 2 V elements: of the rotated part V pairs, else 2 V elements copied.
// The heads of a token in order q, k, v; q goes to q_out, k (rotated) and v to
// the pages (KT = kKvF32 / kKvF16).  Workgroup (x, y): tokens x * T .. and of
// their units the y-th share.  V = 4 needs 16-byte aligned rows, head_dim and
// rot multiples of 8; V = 1 takes any even ones.  2048 tokens of 32 heads of 128
// (67 MB in and out): 11.7 us, 5.7 TB/s, bound by memory; one token of 40 heads
// 2.8 us, with k and v to F16 pages 3.6, bound by the launch and one round trip.
template <int KT, int V>
__global__ __launch_bounds__(256) void rotate_kernel(RotArgs a, int T, int share) {
    extern __shared__ float2 s_cs[];
    const int t0 = blockIdx.x * T, nt = min(T, a.n_tokens - t0);
    const int hd = a.rope.head_dim, half = a.rope.rot / 2, per_head = hd / (2 * V), pairs = half / V;
    const int heads = a.n_head + (KT == kNoPages ? 0 : 2 * a.n_kv), units = heads * per_head;
    const int first = blockIdx.y * share, count = min(share, units - first);
    bool ready = false;
    for (int idx = threadIdx.x; idx < nt * count || !ready; idx += 256) {
        const bool live = idx < nt * count;
        const int t = live ? idx / count : 0, unit = first + (live ? idx - t * count : 0);
        const int h = unit / per_head, u = unit - h * per_head;
        const size_t tok = static_cast<size_t>(t0 + t);
        const bool is_q = h < a.n_head, is_v = KT != kNoPages && h >= a.n_head + a.n_kv;
        const int kh = is_q ? 0 : is_v ? h - a.n_head - a.n_kv : h - a.n_head;
        const float* src = is_q ? a.q + tok * a.q_pitch + static_cast<size_t>(h) * hd
                                : (is_v ? a.v + tok * a.v_pitch : a.k + tok * a.k_pitch) + static_cast<size_t>(kh) * hd;
        const bool turn = u < pairs && !is_v;
        // offsets of the unit's two vectors within the head
        int d0, d1;
        if (turn && a.rope.layout == kRopeHalf) d0 = u * V, d1 = d0 + half;
        else d0 = u * 2 * V, d1 = d0 + V;  // an interleaved unit, or one of the copied part
        Vec<V> x0 = {}, x1 = {};
        if (live) {
            x0 = ld_vec<V>(src + d0);
            x1 = ld_vec<V>(src + d1);
        }
        if (!ready) {
            fill_turns(a, t0, nt, s_cs);
            __syncthreads();
            ready = true;
        }
        if (!live) break;
        if (turn) {
            const float2* cs = s_cs + t * half + u * V;
            Vec<V> y0, y1;
            if (a.rope.layout == kRopeHalf) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 c = cs[j];
                    y0.f[j] = x0.f[j] * c.x - x1.f[j] * c.y;
                    y1.f[j] = x0.f[j] * c.y + x1.f[j] * c.x;
                }
            } else if constexpr (V == 1) {
                const float2 c = cs[0];
                y0.f[0] = x0.f[0] * c.x - x1.f[0] * c.y;
                y1.f[0] = x0.f[0] * c.y + x1.f[0] * c.x;
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const float2 c = cs[j / 2], e = cs[V / 2 + j / 2];
                    y0.f[j] = x0.f[j] * c.x - x0.f[j + 1] * c.y;
                    y0.f[j + 1] = x0.f[j] * c.y + x0.f[j + 1] * c.x;
                    y1.f[j] = x1.f[j] * e.x - x1.f[j + 1] * e.y;
                    y1.f[j + 1] = x1.f[j] * e.y + x1.f[j + 1] * e.x;
                }
            }
            x0 = y0;
            x1 = y1;
        }
        if (is_q) {
            float* dst = a.q_out + tok * a.out_pitch + static_cast<size_t>(h) * hd;
            st_vec<V>(dst + d0, x0);
            st_vec<V>(dst + d1, x1);
        } else if constexpr (KT != kNoPages) {
            const int p = a.pos + t0 + t;
            void* page = (is_v ? a.pt_v : a.pt_k)[p / a.page_tokens];
            const size_t off = static_cast<size_t>(p % a.page_tokens) * a.kv_dim + static_cast<size_t>(kh) * hd;
            if constexpr (KT == kKvF16) {
                st_half<V>(static_cast<uint16_t*>(page) + off + d0, x0);
                st_half<V>(static_cast<uint16_t*>(page) + off + d1, x1);
            } else {
                st_vec<V>(static_cast<float*>(page) + off + d0, x0);
                st_vec<V>(static_cast<float*>(page) + off + d1, x1);
            }
        }
    }
}

// q of the tokens of one group of 8 (workgroup share `part` of `parts`), cs [8][rot / 2] ready.
__device__ __forceinline__ void rotate_q(const RotArgs& a, int t0, int nt, int part, int parts, const float2* cs, bool vec) {
    const int hd = a.rope.head_dim, quads = hd / 4, n = a.n_head * quads, half = a.rope.rot / 2;
    for (int idx = part * blockDim.x + threadIdx.x; idx < nt * n; idx += parts * blockDim.x) {
        const int t = idx / n, r = idx - t * n, h = r / quads, d = (r - h * quads) * 4;
        const size_t tok = static_cast<size_t>(t0 + t), at = static_cast<size_t>(h) * hd;
        const float4 y = rope_quad(a.rope, a.q + tok * a.q_pitch + at, d, cs + t * half, vec);
        float* dst = a.q_out + tok * a.out_pitch + at + d;
        if (vec) {
            *reinterpret_cast<float4*>(dst) = y;
        } else {
            dst[0] = y.x, dst[1] = y.y, dst[2] = y.z, dst[3] = y.w;
        }
    }
}

// A row's four elements e .. e+3, rotated if rope.rot != 0
__device__ __forceinline__ float4 row_quad(const RotArgs& a, const float* row, int e, const float2* cs, bool rot, bool vec) {
    if (!rot) {
        if (vec) return *reinterpret_cast<const float4*>(row + e);
        return make_float4(row[e], row[e + 1], row[e + 2], row[e + 3]);
    }
    const int hd = a.rope.head_dim, h = e / hd;
    return rope_quad(a.rope, row + h * hd, e - h * hd, cs, vec);
}

// Q8 pages: one scale for the whole row, so a workgroup per (token, K or V)
// holds the row in registers as kv_write_q8_kernel does (same rounding, same
// bytes), and workgroups y >= 2 rotate q.  In place q_out == q would race here
// (a quad's pairs belong to two threads): the host takes rotate_kernel for q then.
// Bound by latency (the row's maximum lies between its load and its store): 77
// tokens of 256 channels with 32 heads of 64 of q 4.0 us.
constexpr int kQT = 1024;
constexpr int kQV = 4;
__global__ __launch_bounds__(kQT) void append_q8_kernel(RotArgs a, bool vec) {
    extern __shared__ float2 s_cs[];
    __shared__ float red[kQT / 64];
    const int t = blockIdx.x, which = blockIdx.y;
    const bool rot = which != 1;
    float4 xv[kQV];
    if (rot) {
        fill_turns(a, t, 1, s_cs);
        __syncthreads();
    }
    if (which >= 2) {
        rotate_q(a, t, 1, which - 2, gridDim.y - 2, s_cs, vec);
        return;
    }
    const float* x = which ? a.v + static_cast<size_t>(t) * a.v_pitch : a.k + static_cast<size_t>(t) * a.k_pitch;
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < kQV; ++j) {
        const int d = 4 * (j * kQT + static_cast<int>(threadIdx.x));
        xv[j] = d < a.kv_dim ? row_quad(a, x, d, s_cs, rot, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
        m = fmaxf(m, fmaxf(fmaxf(fabsf(xv[j].x), fabsf(xv[j].y)), fmaxf(fabsf(xv[j].z), fabsf(xv[j].w))));
    }
    m = wave_max_all(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < kQT / 64; ++w) m = fmaxf(m, red[w]);
    const float s = m > 0.0f ? __fdiv_rn(m, 127.0f) : 1.0f;
    const int p = a.pos + t, slot = p % a.page_tokens;
    uint8_t* page = static_cast<uint8_t*>((which ? a.pt_v : a.pt_k)[p / a.page_tokens]);
    int8_t* row = reinterpret_cast<int8_t*>(page) + static_cast<size_t>(slot) * a.kv_dim;
    auto qz = [&](float z) { return static_cast<uint32_t>(static_cast<int>(q_round_away(__fdiv_rn(z, s), 127.0f))) & 0xffu; };
#pragma unroll
    for (int j = 0; j < kQV; ++j) {
        const int d = 4 * (j * kQT + static_cast<int>(threadIdx.x));
        if (d < a.kv_dim)
            *reinterpret_cast<uint32_t*>(row + d) =
                qz(xv[j].x) | (qz(xv[j].y) << 8) | (qz(xv[j].z) << 16) | (qz(xv[j].w) << 24);
    }
    if (threadIdx.x == 0) reinterpret_cast<float*>(page + kv_scale_offset(a.page_tokens, a.kv_dim))[slot] = s;
}

// A quad of a head and what it turns with: loaded first, turned once the turns
// are there.  LAYOUT < 0: no rotation; VEC as in rope_quad.
template <int LAYOUT, bool VEC>
struct TurnQuad {
    float4 own, mate;  // the quad; the one its pairs' other elements are in (half layout)
    int d;
    const float* head;  // the head's first element

    __device__ __forceinline__ void load(const RopeView& r, const float* x, int at) {
        head = x;
        d = at;
        if constexpr (VEC || LAYOUT < 0) {
            const int half = r.rot / 2;
            if constexpr (VEC) own = *reinterpret_cast<const float4*>(x + d);
            else own = make_float4(x[d], x[d + 1], x[d + 2], x[d + 3]);
            if constexpr (LAYOUT == kRopeHalf) mate = *reinterpret_cast<const float4*>(x + (d >= r.rot ? d : d < half ? d + half : d - half));
        }
    }
    __device__ __forceinline__ float4 turned(const RopeView& r, const float2* cs) const {
        if constexpr (LAYOUT < 0) return own;
        if constexpr (!VEC) return rope_quad(r, head, d, cs, false);
        if (d >= r.rot) return own;
        const float x[4] = {own.x, own.y, own.z, own.w};
        float y[4];
        if constexpr (LAYOUT == kRopeHalf) {
            const int half = r.rot / 2;
            const bool low = d < half;
            const float m[4] = {mate.x, mate.y, mate.z, mate.w}, sgn = low ? -1.0f : 1.0f;
            const float2* t = cs + (low ? d : d - half);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = x[j] * t[j].x + sgn * (m[j] * t[j].y);
        } else {
            const float2 t0 = cs[d / 2], t1 = cs[d / 2 + 1];
            y[0] = x[0] * t0.x - x[1] * t0.y;
            y[1] = x[0] * t0.y + x[1] * t0.x;
            y[2] = x[2] * t1.x - x[3] * t1.y;
            y[3] = x[2] * t1.y + x[3] * t1.x;
        }
        return make_float4(y[0], y[1], y[2], y[3]);
    }
};

// The codes, step and middle of a block of 32 held as four elements in each of
// 8 lanes.  Divisions by the format's definition: range / 15 in double (a
// 24-bit number over 15 is no closer to a rounding border than 2^-29 of it, so
// one rounding of the double product is the correct one); (x - c) / s as a
// product with 1 / s, off by 2^-22 of it, and by division itself only where
// that is within 4e-6 of a border between two codes (1 in 10^5 elements).
struct Q4Quad {
    uint32_t code[4];
    uint16_t step, middle;
};
__device__ __forceinline__ Q4Quad quantize_q4_x4(float4 v) {
    const float f[4] = {v.x, v.y, v.z, v.w};
    float mn = fminf(fminf(f[0], f[1]), fminf(f[2], f[3])), mx = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
    float bad = fmaf(f[0], 0.0f, fmaf(f[1], 0.0f, fmaf(f[2], 0.0f, f[3] * 0.0f)));  // 0, or NaN
    mn = -group_max<8>(-mn);
    mx = group_max<8>(mx);
    bad = bad + dpp_mov<0xb1>(bad);
    bad = bad + dpp_mov<0x4e>(bad);
    bad = bad + dpp_mov<0x141>(bad);
    const float fifteenth = static_cast<float>(static_cast<double>(mx - mn) * (1.0 / 15.0));
    const _Float16 s16 = static_cast<_Float16>(fminf(fifteenth, kQ4MaxStep));
    const float s = static_cast<float>(s16);
    const _Float16 c16 = static_cast<_Float16>(fminf(fmaxf(fmaf(8.0f, s, mn), -65504.0f), 65504.0f));
    const float c = static_cast<float>(c16), inv = __builtin_amdgcn_rcpf(s);
    float n[4];
    bool near = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float q = (f[j] - c) * inv;
        n[j] = __builtin_rintf(q);
        near = near || fabsf(q - n[j]) > 0.5f - 4.0e-6f;
    }
    if (__any(near && s > 0.0f)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) n[j] = __builtin_rintf(__fdiv_rn(f[j] - c, s));
    }
    Q4Quad r;
    const bool fine = s > 0.0f && bad == 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        r.code[j] = fine ? static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(n[j] + 8.0f, 0.0f), 15.0f))) : 8u;
    r.step = bad == 0.0f ? __builtin_bit_cast(uint16_t, s16) : static_cast<uint16_t>(0x7e00);
    r.middle = bad == 0.0f ? __builtin_bit_cast(uint16_t, c16) : static_cast<uint16_t>(0);
    return r;
}

// Q4 pages (layout and rounding: mvh_kv4.hpp).  Workgroup (x, y): the x-th
// group of 8 rows that the call touches; y < kv_parts a share of the K blocks,
// then of the V blocks, then of q (a token's heads in q_parts shares).  A wave
// takes two blocks at a time: lane = (row i, four channels), the block's
// minimum and maximum by DPP over 8 lanes.  A V word holds the group's 8 rows
// of a channel: rows of the group that this call does not write keep their
// nibbles (the word is this wave's alone).  512 tokens of 1024 channels with 32
// heads of 128 of q (26 MB in and out): 6.9 us, 3.7 TB/s, VALU 31 % busy.
constexpr int kA4 = 256;
template <int LAYOUT, bool VEC>
__global__ __launch_bounds__(kA4) void append_q4_kernel(RotArgs a, Kv4Map map, int kv_parts, int q_parts, uint64_t hd_recip,
                                                        const int* d_pos) {
    extern __shared__ float2 s_cs[];
    a.pos = d_pos ? *d_pos : a.pos;
    const int vg = map.group_of(a.pos) + blockIdx.x, page = map.page_of(vg), g = vg - page * map.groups;
    const int row0 = page * map.page_tokens + g * 8;  // position of the group's first row
    const int lo = max(a.pos - row0, 0);
    const int hi = min(min(a.pos + a.n_tokens - row0, 8), map.page_tokens - g * 8);  // rows lo .. hi-1 are written
    if (lo >= hi) return;  // a device position that starts later in its group than the grid allows for
    const int t0 = row0 + lo - a.pos;  // token of row lo
    const int half = a.rope.rot / 2, hd = a.rope.head_dim;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, nblk = a.kv_dim / 32;
    const int part = blockIdx.y;
    if constexpr (LAYOUT >= 0) {
        if (part >= 2 * kv_parts) {  // a token's q heads: a thread keeps its quad of the head
            const int p = part - 2 * kv_parts, t = p / q_parts, hp = p - t * q_parts;
            if (t >= hi - lo) return;
            const int quads = hd / 4, per = kA4 / quads, h0 = threadIdx.x / quads, d = (threadIdx.x - h0 * quads) * 4;
            const float* x = a.q + static_cast<size_t>(t0 + t) * a.q_pitch;
            float* y = a.q_out + static_cast<size_t>(t0 + t) * a.out_pitch + d;
            int h = h0 + hp * per;
            const bool live = h0 < per;
            TurnQuad<LAYOUT, VEC> quad;
            if (live && h < a.n_head) quad.load(a.rope, x + static_cast<size_t>(h) * hd, d);
            fill_turns(a, t0 + t, 1, s_cs);
            __syncthreads();
            while (live && h < a.n_head) {
                const float4 v = quad.turned(a.rope, s_cs);
                float* dst = y + static_cast<size_t>(h) * hd;
                h += per * q_parts;
                if (h < a.n_head) quad.load(a.rope, x + static_cast<size_t>(h) * hd, d);
                if constexpr (VEC) {
                    *reinterpret_cast<float4*>(dst) = v;
                } else {
                    dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
                }
            }
            return;
        }
    }
    const bool is_v = part >= kv_parts;
    const int i = lane >> 3, c4 = lane & 7;
    const bool live = i >= lo && i < hi;
    const int tok = t0 + (live ? i - lo : 0), step = kv_parts * (kA4 / 64);
    uint8_t* const base = static_cast<uint8_t*>((is_v ? a.pt_v : a.pt_k)[page]);
    uint8_t* const nibbles = base + static_cast<size_t>(g) * 128;
    uint16_t* const scales = reinterpret_cast<uint16_t*>(base + kv4_scales(map.page_tokens, a.kv_dim) + static_cast<size_t>(g) * 32) + kv4_scale(i);
    const size_t n_blk = static_cast<size_t>(map.groups) * 128, s_blk = static_cast<size_t>(map.groups) * 16;
    int b = (is_v ? part - kv_parts : part) * (kA4 / 64) + wave;
    auto put_scales = [&](int blk, const Q4Quad& q) {
        if (live && c4 == 0) {
            scales[blk * s_blk] = q.step;
            scales[blk * s_blk + 8] = q.middle;
        }
    };
    if (!is_v) {
        const float* x = a.k + static_cast<size_t>(tok) * a.k_pitch;
        TurnQuad<LAYOUT, VEC> quad[2];
        auto load = [&](int blk, TurnQuad<LAYOUT, VEC>& q) {
            const int e = blk * 32 + 4 * c4;
            if constexpr (LAYOUT < 0) {
                q.load(a.rope, x, e);
            } else {
                const int h = static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(e)) * hd_recip) >> 40);
                q.load(a.rope, x + h * hd, e - h * hd);
            }
        };
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (b + u * step < nblk) load(b + u * step, quad[u]);
        if constexpr (LAYOUT >= 0) {
            fill_turns(a, t0, hi - lo, s_cs);
            __syncthreads();
        }
        const float2* cs = s_cs + (live ? i - lo : 0) * half;
        for (; b < nblk; b += 2 * step) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int blk = b + u * step;
                if (blk >= nblk) break;
                const Q4Quad q = quantize_q4_x4(quad[u].turned(a.rope, cs));
                if (blk + 2 * step < nblk) load(blk + 2 * step, quad[u]);
                put_scales(blk, q);
                const uint32_t own = q.code[0] | (q.code[1] << 4) | (q.code[2] << 8) | (q.code[3] << 12);
                const uint32_t mate = static_cast<uint32_t>(dpp_mov<0xb1>(static_cast<int>(own)));
                if (live && !(c4 & 1)) reinterpret_cast<uint32_t*>(nibbles + blk * n_blk)[kv4_k_word(i, c4 >> 1)] = kv4_store(own | (mate << 16));
            }
        }
        return;
    }
    const float* x = a.v + static_cast<size_t>(tok) * a.v_pitch;
    const uint32_t mask = ~((hi == 8 ? 0u : 0xffffffffu << (4 * hi)) | ((1u << (4 * lo)) - 1u));  // the nibbles it writes
    const int ch = 4 * c4 + (i & 3), word = kv4_v_word(ch);  // the channel whose word lanes i < 4 write
    const uint32_t pick = (i & 3) | ((4 + (i & 3)) << 8);
    TurnQuad<-1, VEC> quad[2];
    uint32_t old[2] = {0u, 0u};
    auto load = [&](int blk, int u) {
        quad[u].load(a.rope, x, blk * 32 + 4 * c4);
        if (mask != 0xffffffffu && i < 4) old[u] = reinterpret_cast<const uint32_t*>(nibbles + blk * n_blk)[word];
    };
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (b + u * step < nblk) load(b + u * step, u);
    for (; b < nblk; b += 2 * step) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int blk = b + u * step;
            if (blk >= nblk) break;
            const Q4Quad q = quantize_q4_x4(quad[u].own);
            const uint32_t kept = kv4_nat(old[u]) & ~mask;
            if (blk + 2 * step < nblk) load(blk + 2 * step, u);
            put_scales(blk, q);
            // 8 rows of 4 channels turned into 4 words: two rows a byte (lanes 8 on), then rows 2 and 3, 4 to 7 (16, 32 on)
            uint32_t p = q.code[0] | (q.code[1] << 8) | (q.code[2] << 16) | (q.code[3] << 24);
            p = live ? p << (4 * (i & 1)) : 0u;
            p |= static_cast<uint32_t>(dpp_mov<0x128>(static_cast<int>(p)));
            const auto r16 = __builtin_amdgcn_permlane16_swap(p, p, false, false);
            const auto ra = __builtin_amdgcn_permlane32_swap(r16[0], r16[0], false, false);
            const auto rb = __builtin_amdgcn_permlane32_swap(r16[1], r16[1], false, false);
            const uint32_t w_lo = __builtin_amdgcn_perm(rb[0], ra[0], pick), w_hi = __builtin_amdgcn_perm(rb[1], ra[1], pick);
            const uint32_t nat = __builtin_amdgcn_perm(w_hi, w_lo, 0x05040100u);
            if (i < 4) reinterpret_cast<uint32_t*>(nibbles + blk * n_blk)[word] = kv4_store(kept | nat);
        }
    }
}

// Rows pos .. of K (y = 0) or V (y = 1) as fp32, four elements a thread: bound by
// the stores (512 rows of 1024 channels from 4 bits 4.2 us, a few rows 2.4).
template <int KT>
__global__ __launch_bounds__(256) void kv_read_kernel(const void* const* __restrict__ pt_k,
                                                      const void* const* __restrict__ pt_v, int pos, int n_tokens,
                                                      int kv_dim, int page_tokens, float* __restrict__ k,
                                                      float* __restrict__ v) {
    const int which = blockIdx.y, quads = kv_dim / 4;
    float* out = which ? v : k;
    if (!out) return;
    const size_t idx = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    const size_t t = idx / quads;
    if (t >= static_cast<size_t>(n_tokens)) return;
    const int e = static_cast<int>(idx - t * quads) * 4, p = pos + static_cast<int>(t), slot = p % page_tokens;
    const uint8_t* page = static_cast<const uint8_t*>((which ? pt_v : pt_k)[p / page_tokens]);
    float f[4];
    if constexpr (KT == kKvQ4) {
        const int groups = static_cast<int>(kv4_groups(page_tokens)), b = e / 32, ch = e % 32, g = slot / 8, i = slot % 8;
        const size_t at = static_cast<size_t>(b) * groups + g;
        const uint8_t* sc = page + kv4_scales(page_tokens, kv_dim) + at * 32;
        const float s = kv4_step(sc, i), c = kv4_middle(sc, i);
        const uint32_t* words = reinterpret_cast<const uint32_t*>(page + at * 128);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t n = which ? kv4_nat(words[kv4_v_word(ch + j)]) >> (4 * i)
                                     : kv4_nat(words[kv4_k_word(i, ch / 8)]) >> (4 * (ch % 8 + j));
            f[j] = s * (static_cast<float>(n & 15u) - 8.0f) + c;
        }
    } else {
        const void* row = page + static_cast<size_t>(slot) * kv_dim * kv_elem_bytes(KT);
        const float sc = kv_row_scale<KT>(page, slot, page_tokens, kv_dim);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = kv_to_f<KT>(row, e + j);
            if constexpr (KT == kKvQ8) f[j] *= sc;
        }
    }
    float* dst = out + t * kv_dim + e;
    if ((reinterpret_cast<uintptr_t>(out) & 15) == 0) {
        *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        dst[0] = f[0], dst[1] = f[1], dst[2] = f[2], dst[3] = f[3];
    }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int KT>
hipError_t rotate_typed(const RotArgs& a, hipStream_t st) {
    const int hd = a.rope.head_dim, rot = a.rope.rot, heads = a.n_head + (KT == kNoPages ? 0 : 2 * a.n_kv);
    bool vec = hd % 8 == 0 && rot % 8 == 0;
    if (a.n_head) vec = vec && al16(a.q) && al16(a.q_out) && a.q_pitch % 4 == 0 && a.out_pitch % 4 == 0;
    if (KT != kNoPages) vec = vec && al16(a.k) && al16(a.v) && a.k_pitch % 4 == 0 && a.v_pitch % 4 == 0;
    const int units = heads * (hd / (vec ? 8 : 2));
    // several tokens a workgroup while they fit 256 threads (and 32 KB of turns); else a token's units in shares
    const int T = std::max(1, std::min({256 / units, a.n_tokens, 4096 / std::max(1, rot / 2)}));
    const int share = T > 1 ? units : std::max(std::min(units, a.n_tokens >= 512 ? 512 : 256), (units + 65534) / 65535);
    const dim3 grid(static_cast<unsigned>((a.n_tokens + T - 1) / T), static_cast<unsigned>((units + share - 1) / share));
    const size_t lds = static_cast<size_t>(T) * (rot / 2) * sizeof(float2);
    if (vec) rotate_kernel<KT, 4><<<grid, 256, lds, st>>>(a, T, share);
    else rotate_kernel<KT, 1><<<grid, 256, lds, st>>>(a, T, share);
    return hipGetLastError();
}

template <int LAYOUT, bool VEC>
hipError_t append_q4(const RotArgs& a, const int* d_pos, hipStream_t st) {
    const Kv4Map map = kv4_map(a.page_tokens);
    const int groups = d_pos ? 1 : map.group_of(a.pos + a.n_tokens - 1) - map.group_of(a.pos) + 1;
    const int nblk = a.kv_dim / 32, rows = std::min(8, a.n_tokens);
    // a wave two blocks, or one where the chip has room for that (few rows: the shortest path counts)
    const int per = groups * nblk >= 2048 ? 8 : 4, kv_parts = (nblk + per - 1) / per;
    int q_parts = 0;
    uint64_t recip = 0;
    if constexpr (LAYOUT >= 0) {
        const int heads_at_once = kA4 / (a.rope.head_dim / 4);
        if (a.n_head) q_parts = std::max(1, (a.n_head + 4 * heads_at_once - 1) / (4 * heads_at_once));
        recip = (uint64_t{1} << 40) / static_cast<uint64_t>(a.rope.head_dim) + 1;  // exact below 2^16 elements, heads up to 2^10
    }
    const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(2 * kv_parts + rows * q_parts));
    const size_t lds = LAYOUT >= 0 ? rows * (a.rope.rot / 2) * sizeof(float2) : 0;
    append_q4_kernel<LAYOUT, VEC><<<grid, kA4, lds, st>>>(a, map, kv_parts, q_parts, recip, d_pos);
    return hipGetLastError();
}

RopeView no_rope() { return RopeView{}; }

constexpr size_t kMostTokens = size_t{1} << 22;  // of a launch of rotate_kernel
constexpr size_t kMostQuads = size_t{1} << 31;   // of a launch of kv_read_kernel, a thread each

}  // namespace

hipError_t launch_rope(const RopeView& rope, const float* x, size_t x_pitch, float* out, size_t out_pitch,
                       const int* positions, size_t pos, size_t n_tokens, size_t n_head, hipStream_t st) {
    if (!n_tokens || !n_head) return hipSuccess;
    RotArgs a{};
    a.rope = rope;
    a.q_pitch = x_pitch;
    a.out_pitch = out_pitch;
    a.n_head = static_cast<int>(n_head);
    // a workgroup a token at worst: launches of 2^22 tokens stay below the 2^32 threads a grid may have
    for (size_t t = 0; t < n_tokens; t += kMostTokens) {
        a.q = x + t * x_pitch;
        a.q_out = out + t * out_pitch;
        a.positions = positions ? positions + t : nullptr;
        a.pos = static_cast<int>(pos + t);
        a.n_tokens = static_cast<int>(std::min(n_tokens - t, kMostTokens));
        if (hipError_t e = rotate_typed<kNoPages>(a, st); e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_kv_append(int kv_type, const RopeView& rope, void* const* pt_k, void* const* pt_v, const float* q,
                            size_t q_pitch, float* q_out, size_t out_pitch, const float* k, size_t k_pitch,
                            const float* v, size_t v_pitch, size_t pos, size_t n_tokens, size_t n_head, size_t kv_dim,
                            size_t page_tokens, hipStream_t st) {
    if (!n_tokens) return hipSuccess;
    RotArgs a{};
    a.rope = rope;
    a.q = q;
    a.q_out = q_out;
    a.k = k;
    a.v = v;
    a.q_pitch = q_pitch;
    a.out_pitch = out_pitch;
    a.k_pitch = k_pitch;
    a.v_pitch = v_pitch;
    a.pos = static_cast<int>(pos);
    a.n_tokens = static_cast<int>(n_tokens);
    a.n_head = static_cast<int>(n_head);
    a.n_kv = static_cast<int>(kv_dim / rope.head_dim);
    a.pt_k = pt_k;
    a.pt_v = pt_v;
    a.page_tokens = static_cast<int>(page_tokens);
    a.kv_dim = static_cast<int>(kv_dim);
    if (kv_type == kKvF32) return rotate_typed<kKvF32>(a, st);
    if (kv_type == kKvF16) return rotate_typed<kKvF16>(a, st);
    // the quads of q are read and written by different threads: in place, q goes through a launch of its own
    if (a.n_head && q == q_out) {
        if (hipError_t e = launch_rope(rope, q, q_pitch, q_out, out_pitch, nullptr, pos, n_tokens, n_head, st); e != hipSuccess)
            return e;
        a.n_head = 0;
    }
    bool vec = rope.layout == kRopeHalf ? rope.rot % 8 == 0 : rope.rot % 4 == 0;
    vec = vec && al16(k) && al16(v) && k_pitch % 4 == 0 && v_pitch % 4 == 0;
    if (a.n_head) vec = vec && al16(q) && al16(q_out) && q_pitch % 4 == 0 && out_pitch % 4 == 0;
    const size_t q_quads = static_cast<size_t>(a.n_head) * rope.head_dim / 4;
    if (kv_type == kKvQ8) {
        if (kv_dim > 4 * kQT * kQV) return hipErrorInvalidValue;
        const unsigned parts = a.n_head ? static_cast<unsigned>((q_quads + kQT - 1) / kQT) : 0;
        append_q8_kernel<<<dim3(static_cast<unsigned>(n_tokens), 2 + parts), kQT, rope.rot / 2 * sizeof(float2), st>>>(a, vec);
        return hipGetLastError();
    }
    if (kv_type != kKvQ4) return hipErrorInvalidValue;
    const int layout = rope.layout;
    if (vec) return layout == kRopeHalf ? append_q4<kRopeHalf, true>(a, nullptr, st) : append_q4<kRopeInterleaved, true>(a, nullptr, st);
    return layout == kRopeHalf ? append_q4<kRopeHalf, false>(a, nullptr, st) : append_q4<kRopeInterleaved, false>(a, nullptr, st);
}

hipError_t launch_kv4_write(void* const* pt_k, void* const* pt_v, const float* k, const float* v, size_t pitch,
                            const int* d_pos, size_t pos, size_t n_tokens, size_t kv_dim, size_t page_tokens,
                            hipStream_t st) {
    if (!n_tokens) return hipSuccess;
    if (kv_dim % 32 || (d_pos && n_tokens != 1)) return hipErrorInvalidValue;
    RotArgs a{};
    a.rope = no_rope();
    a.k = k;
    a.v = v;
    a.k_pitch = a.v_pitch = pitch;
    a.pos = static_cast<int>(pos);
    a.n_tokens = static_cast<int>(n_tokens);
    a.pt_k = pt_k;
    a.pt_v = pt_v;
    a.page_tokens = static_cast<int>(page_tokens);
    a.kv_dim = static_cast<int>(kv_dim);
    const bool vec = al16(k) && al16(v) && pitch % 4 == 0;
    return vec ? append_q4<-1, true>(a, d_pos, st) : append_q4<-1, false>(a, d_pos, st);
}

hipError_t launch_kv_read(int kv_type, const void* const* pt_k, const void* const* pt_v, size_t pos, size_t n_tokens,
                          size_t kv_dim, size_t page_tokens, float* k, float* v, hipStream_t st) {
    const size_t quads = kv_dim / 4, most = std::max<size_t>(1, kMostQuads / quads);
    for (size_t t = 0; t < n_tokens; t += most) {
        const size_t rows = std::min(n_tokens - t, most);
        const dim3 grid(static_cast<unsigned>((rows * quads + 255) / 256), 2);
        const int p = static_cast<int>(pos + t), n = static_cast<int>(rows), kd = static_cast<int>(kv_dim),
                  pt = static_cast<int>(page_tokens);
        float *kt = k ? k + t * kv_dim : nullptr, *vt = v ? v + t * kv_dim : nullptr;
        switch (kv_type) {
        case kKvF32: kv_read_kernel<kKvF32><<<grid, 256, 0, st>>>(pt_k, pt_v, p, n, kd, pt, kt, vt); break;
        case kKvF16: kv_read_kernel<kKvF16><<<grid, 256, 0, st>>>(pt_k, pt_v, p, n, kd, pt, kt, vt); break;
        case kKvQ8: kv_read_kernel<kKvQ8><<<grid, 256, 0, st>>>(pt_k, pt_v, p, n, kd, pt, kt, vt); break;
        case kKvQ4: kv_read_kernel<kKvQ4><<<grid, 256, 0, st>>>(pt_k, pt_v, p, n, kd, pt, kt, vt); break;
        default: return hipErrorInvalidValue;
        }
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mvh
