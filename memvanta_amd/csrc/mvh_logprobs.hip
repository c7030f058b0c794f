// mvh_logprobs.hip -- log probabilities of a row of logits: of a given token,
// the entropy, and the most probable tokens.
//
// One pass over the row with a running maximum m:
//   s = sum e^(l - m), t = sum (l - m) e^(l - m),
//   log p_i = (l_i - m) - ln s,  entropy = ln s - t / s,
// all in fp32 per thread, joined across threads with the usual rescaling.  The
// pass is bound by reading the logits (~10 operations an element); few
// rows of more than 65536 are cut into parts, whose sums and candidates a second
// kernel joins.
//
// The most probable tokens, a tile of the row (32 elements a lane) at a time:
// the k-th of the largest elements of 64 groups of lanes is a bound that at
// least k elements reach, and few more (24 of 32000 random ones for k = 20);
// what reaches it is set aside in LDS, sorted by value, then index, by the waves
// 64 at a time, and merged by one into the best 64 so far.  In later tiles the
// bound is the k-th best so far.  Where too many are equal (a row with fewer
// unmasked tokens than k, or than there are groups that hold one) every wave
// sorts its own elements 64 at a time instead, three to four times as long (one row
// of 32000 with 64 tops 12.3 us, 42 with 32 tokens left; 768 rows with 20 tops 29
// and 114).
#include "mvh_kernels.hpp"

#include <type_traits>

namespace mvh {
namespace {

constexpr int kPer = 32;  // elements a lane holds at once
constexpr int kSetAside = 1024;  // candidates of a tile that have room
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFar = -1.0e4f;  // e^kFar is 0; keeps 0 * (l - m) from being 0 * inf

// lane ^ X of a wave, by lane moves (no LDS round trip)
template <int X>
__device__ __forceinline__ int lane_xor(int v, int lane) {
    if constexpr (X == 1) return dpp_mov<0xb1>(v);
    else if constexpr (X == 2) return dpp_mov<0x4e>(v);
    else if constexpr (X == 4) return dpp_mov<0x1b>(dpp_mov<0x141>(v));  // ^ 7, then ^ 3
    else if constexpr (X == 8) return dpp_mov<0x128>(v);                 // 8 on within 16
    else if constexpr (X == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return static_cast<int>(lane & 16 ? r[0] : r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return static_cast<int>(lane & 32 ? r[0] : r[1]);
    }
}
template <int X>
__device__ __forceinline__ float lane_xor(float v, int lane) {
    return __int_as_float(lane_xor<X>(__float_as_int(v), lane));
}

struct Sums {
    float m, s, t;
};

// b's sums joined into a's
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    const float da = fmaxf(a.m - m, kFar), db = fmaxf(b.m - m, kFar);
    const float ra = __builtin_amdgcn_exp2f((a.m - m) * kLog2e), rb = __builtin_amdgcn_exp2f((b.m - m) * kLog2e);
    return {m, fmaf(a.s, ra, b.s * rb), fmaf(ra, fmaf(da, a.s, a.t), rb * fmaf(db, b.s, b.t))};
}
template <int X>
__device__ __forceinline__ Sums join_xor(Sums a, int lane) {
    return join(a, Sums{lane_xor<X>(a.m, lane), lane_xor<X>(a.s, lane), lane_xor<X>(a.t, lane)});
}
__device__ __forceinline__ Sums wave_join(Sums a, int lane) {
    a = join_xor<8>(join_xor<4>(join_xor<2>(join_xor<1>(a, lane), lane), lane), lane);
    return join_xor<32>(join_xor<16>(a, lane), lane);
}

typedef unsigned long long u64;

// larger value first, then lower index; -0 and +0 are equal
__device__ __forceinline__ u64 key_of(float x, int idx) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t o = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return (static_cast<u64>(o) << 32) | static_cast<uint32_t>(~idx);
}
__device__ __forceinline__ float key_value(u64 k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int key_index(u64 k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

template <int X>
__device__ __forceinline__ u64 key_xor(u64 k, int lane) {
    return (static_cast<u64>(static_cast<uint32_t>(lane_xor<X>(static_cast<int>(k >> 32), lane))) << 32) |
           static_cast<uint32_t>(lane_xor<X>(static_cast<int>(k), lane));
}
// lane's key, or the same of float maxima: the element of a compared pair that comes first or last
__device__ __forceinline__ u64 lesser(u64 a, u64 b, bool less) { return less == (b < a) ? b : a; }
__device__ __forceinline__ float lesser(float a, float b, bool less) { return less ? fminf(a, b) : fmaxf(a, b); }
template <int X>
__device__ __forceinline__ u64 other(u64 k, int lane) { return key_xor<X>(k, lane); }
template <int X>
__device__ __forceinline__ float other(float k, int lane) { return lane_xor<X>(k, lane); }

// bitonic steps X, X/2 .. 1 of blocks of SIZE lanes
template <int SIZE, int X, typename T>
__device__ __forceinline__ T sort_steps(T k, int lane) {
    k = lesser(k, other<X>(k, lane), !(lane & X) == !(lane & SIZE));
    if constexpr (X > 1) k = sort_steps<SIZE, X / 2>(k, lane);
    return k;
}
// 64 values, one a lane, sorted ascending (lane 0 the smallest)
template <typename T>
__device__ __forceinline__ T sort_ascending(T k, int lane) {
    k = sort_steps<2, 1>(k, lane);
    k = sort_steps<4, 2>(k, lane);
    k = sort_steps<8, 4>(k, lane);
    k = sort_steps<16, 8>(k, lane);
    k = sort_steps<32, 16>(k, lane);
    return sort_steps<64, 32>(k, lane);
}
template <int X>
__device__ __forceinline__ u64 merge_steps(u64 k, int lane) {
    k = lesser(k, key_xor<X>(k, lane), (lane & X) != 0);
    if constexpr (X > 1) k = merge_steps<X / 2>(k, lane);
    return k;
}
// best (descending) and more (ascending): the best 64 of both, descending
__device__ __forceinline__ u64 merge_best(u64 best, u64 more, int lane) { return merge_steps<32>(best > more ? best : more, lane); }
__device__ __forceinline__ u64 key_reversed(u64 k, int lane) {  // lane 63 - l's
    return (static_cast<u64>(static_cast<uint32_t>(__shfl(static_cast<int>(k >> 32), 63 - lane))) << 32) |
           static_cast<uint32_t>(__shfl(static_cast<int>(k), 63 - lane));
}
__device__ __forceinline__ u64 key_at(u64 k, int lane) {  // lane: the same in every lane
    return (static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k >> 32), lane))) << 32) |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k), lane));
}

// A wave's best k so far, and the candidates set aside for it.
struct Best {
    u64 best = 0, least = 0;  // lane's key of the sorted list; the k-th best (0 while there are fewer)
    int waiting = 0;
    u64* buf;  // 128 keys of LDS, this wave's
    int lane, k;

    __device__ __forceinline__ void flush() {
        __builtin_amdgcn_wave_barrier();
        const u64 c = lane < waiting ? buf[lane] : 0;
        const u64 rest = lane + 64 < waiting ? buf[lane + 64] : 0;
        best = merge_best(best, sort_ascending(c, lane), lane);
        least = key_at(best, k - 1);
        __builtin_amdgcn_wave_barrier();
        if (lane + 64 < waiting) buf[lane] = rest;
        waiting = max(waiting - 64, 0);
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void offer(u64 key) {  // key 0: none
        const bool take = key > least;
        const u64 votes = __ballot(take);
        if (!votes) return;
        const int at = waiting + __popcll(votes & ((u64{1} << lane) - 1));
        if (take) buf[at] = key;
        waiting += __popcll(votes);
        if (waiting >= 64) flush();
    }
};

struct LpArgs {
    const float* logits;
    const int* targets;
    float* logprob;
    float* entropy;
    int* top_ids;
    float* top_lp;
    size_t n, pitch;
    int k, parts;
    size_t chunk;     // elements of a part
    float* part_sums; // [row][part][3]
    u64* part_keys;   // [row][part][64]
};

struct __attribute__((packed, aligned(4))) Quad {
    float f[4];
};

// What the row's results are, from its sums and its best keys (one a lane of one wave)
template <bool TOP>
__device__ __forceinline__ void write_row(const LpArgs& a, size_t row, Sums r, u64 best, int lane) {
    // no finite logit at all: every token has probability 0
    const bool empty = r.s == 0.0f;
    const float ln_s = logf(r.s);
    if (lane == 0) {
        if (a.logprob) {
            const int id = a.targets[row];
            float lp = __builtin_nanf("");
            if (id >= 0 && static_cast<size_t>(id) < a.n)
                lp = empty ? -INFINITY : (a.logits[row * a.pitch + id] - r.m) - ln_s;
            a.logprob[row] = lp;
        }
        if (a.entropy) a.entropy[row] = empty ? 0.0f : ln_s - __fdiv_rn(r.t, r.s);
    }
    if constexpr (TOP) {
        if (lane < a.k) {
            const size_t at = row * a.k + lane;
            // no key: a row with NaN, whose ids are any
            if (a.top_ids) a.top_ids[at] = best ? key_index(best) : lane;
            if (a.top_lp) a.top_lp[at] = empty ? -INFINITY : (key_value(best) - r.m) - ln_s;
        }
    }
}

// A workgroup: one part of a row, tile by tile; a thread takes every NT-th quad of a tile.  In the first tile wave 0
// looks for the bound while the others form their sums, and forms its own while wave kKeyWave sorts what was set
// aside (one row of 32000 logits, 20 tops: 9.0 us, with each step after the other 9.1).
constexpr int kKeyWave = 1;
template <int NT, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_kernel(LpArgs a) {
    constexpr int NW = NT / 64, TILE = NT * kPer, KEYS = TOP ? (NW * 128 > kSetAside ? NW * 128 : kSetAside) : 1;
    __shared__ u64 s_key[KEYS];
    __shared__ float s_top[64];
    __shared__ float s_bound;
    __shared__ int s_count[2];  // of even and odd tiles
    __shared__ Sums s_sums[NW];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const size_t row = blockIdx.y, begin = blockIdx.x * a.chunk, end = min(begin + a.chunk, a.n);
    const float* x = a.logits + row * a.pitch;
    Sums r = {-3.402823466e38f, 0.0f, 0.0f};
    u64 best = 0;  // key wave: the best 64 so far, descending
    float v[kPer], w[NT == 256 ? kPer : 1];
    auto load = [&](size_t at, float* d) {
#pragma unroll
        for (int c = 0; c < kPer / 4; ++c) {
            const size_t i = at + c * (4 * NT);
            if (i + 4 <= end) {
                const Quad q = *reinterpret_cast<const Quad*>(x + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) d[4 * c + j] = q.f[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) d[4 * c + j] = i + j < end ? x[i + j] : -INFINITY;
            }
        }
    };
    size_t at = begin + threadIdx.x * 4;
    load(at, v);
    if (TOP && threadIdx.x == 0) s_count[0] = 0;
    int odd = 0;
    for (size_t tile = begin; tile < end; tile += TILE, at += TILE) {  // the same number of turns for every wave
        const bool more = tile + TILE < end, first = tile == begin;
        if constexpr (NT == 256) {
            if (more) load(at + TILE, w);
        }
        float quad[kPer / 4];
#pragma unroll
        for (int c = 0; c < kPer / 4; ++c) quad[c] = fmaxf(fmaxf(v[4 * c], v[4 * c + 1]), fmaxf(v[4 * c + 2], v[4 * c + 3]));
        float top = quad[0];
#pragma unroll
        for (int c = 1; c < kPer / 4; ++c) top = fmaxf(top, quad[c]);
        auto sums = [&] {
            const float m = fmaxf(r.m, top), dm = fmaxf(r.m - m, kFar), f = __builtin_amdgcn_exp2f(dm * kLog2e);
            float s = r.s * f, t = f * fmaf(dm, r.s, r.t);
    #pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const float d = v[i] - m, p = __builtin_amdgcn_exp2f(d * kLog2e);
                s += p;
                t = fmaf(p, fmaxf(d, kFar), t);
            }
            r = {m, s, t};
        };
        if constexpr (!TOP) sums();
        if constexpr (TOP) {
            float bound;
            if (first) {
                // the largest elements of 64 groups of NW lanes: of these, the k-th
                const float mine = group_max<NW>(fmaxf(top, -INFINITY));
                if (lane % NW == 0) s_top[wave * (64 / NW) + lane / NW] = mine;
                __syncthreads();
                if (wave == 0) {
                    const float all = sort_ascending(s_top[lane], lane);
                    if (lane == 64 - a.k) s_bound = all;
                } else {
                    sums();
                }
                __syncthreads();
                bound = s_bound;
            } else {
                sums();
                bound = s_bound;  // the k-th best so far: later equal ones lose, their index is higher
            }
            // elements of later tiles have to be above it; -inf: fewer than k so far, all are taken
            const bool all_in = first || bound == -INFINITY;
            auto reaches = [&](float f) { return all_in ? f >= bound : f > bound; };
            if (__any(reaches(top))) {
#pragma unroll
                for (int c = 0; c < kPer / 4; ++c) {
                    if (!__any(reaches(quad[c]))) continue;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const size_t i = at + c * (4 * NT) + j;
                        if (reaches(v[4 * c + j]) && i < end) {
                            const int slot = atomicAdd(&s_count[odd], 1);
                            if (slot < kSetAside) s_key[slot] = key_of(v[4 * c + j], static_cast<int>(i));
                        }
                    }
                }
            }
            __syncthreads();
            const int count = s_count[odd];
            if (first && wave == 0) sums();
            if (count <= kSetAside) {
                auto sorted = [&](int c) { return sort_ascending(c + lane < count ? s_key[c + lane] : u64{0}, lane); };
                if (count > 64) {  // 64 a wave
                    for (int c = wave * 64; c < count; c += NT) s_key[c + lane] = sorted(c);
                    __syncthreads();
                }
                if (wave == kKeyWave) {
                    for (int c = 0; c < count; c += 64) {
                        const u64 more_keys = count > 64 ? s_key[c + lane] : sorted(c);
                        best = first && !c ? key_reversed(more_keys, lane) : merge_best(best, more_keys, lane);
                    }
                }
            } else {  // many equal ones
                __syncthreads();
                Best own;
                own.buf = s_key + wave * 128;
                own.lane = lane;
                own.k = a.k;
#pragma unroll 1
                for (int c = 0; c < kPer; ++c) {
                    float vc = v[0];
#pragma unroll
                    for (int i = 1; i < kPer; ++i) vc = c == i ? v[i] : vc;
                    const size_t i = at + (c / 4) * (4 * NT) + c % 4;
                    own.offer(i < end ? key_of(vc, static_cast<int>(i)) : 0);
                }
                while (own.waiting > 0) own.flush();
                __syncthreads();
                s_key[wave * 64 + lane] = own.best;
                __syncthreads();
                if (wave == kKeyWave)
                    for (int k = 0; k < NW; ++k) best = merge_best(best, s_key[k * 64 + 63 - lane], lane);
            }
            if (more) {
                odd ^= 1;
                if (wave == kKeyWave) {
                    const u64 kth = key_at(best, a.k - 1);
                    if (lane == 0) {
                        s_bound = kth ? key_value(kth) : -INFINITY;
                        s_count[odd] = 0;
                    }
                }
                __syncthreads();
            }
        }
        if constexpr (NT == 256) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = w[i];
        } else if (more) {
            load(at + TILE, v);
        }
    }
    r = wave_join(r, lane);
    if (lane == 0) s_sums[wave] = r;
    __syncthreads();
    if (wave != (TOP ? kKeyWave : 0)) return;
    r = lane < NW ? s_sums[lane] : Sums{-3.402823466e38f, 0.0f, 0.0f};
    r = join_xor<2>(join_xor<1>(r, lane), lane);
    if constexpr (NW > 4) r = join_xor<8>(join_xor<4>(r, lane), lane);
    auto lane0 = [](float f) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(f))); };
    r = {lane0(r.m), lane0(r.s), lane0(r.t)};
    if (a.parts == 1) {
        write_row<TOP>(a, row, r, best, lane);
        return;
    }
    const size_t part = row * a.parts + blockIdx.x;
    if (lane == 0) {
        a.part_sums[3 * part] = r.m;
        a.part_sums[3 * part + 1] = r.s;
        a.part_sums[3 * part + 2] = r.t;
    }
    if constexpr (TOP) a.part_keys[64 * part + lane] = best;
}

// A row's parts joined: one wave.
template <bool TOP>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LpArgs a) {
    const size_t row = blockIdx.x;
    const int lane = threadIdx.x;
    Sums r = {-3.402823466e38f, 0.0f, 0.0f};
    for (int p = lane; p < a.parts; p += 64) {
        const float* q = a.part_sums + 3 * (row * a.parts + p);
        r = join(r, Sums{q[0], q[1], q[2]});
    }
    r = wave_join(r, lane);
    u64 best = 0;
    if constexpr (TOP) {
        const u64* keys = a.part_keys + 64 * row * a.parts;
        best = keys[lane];
        for (int p = 1; p < a.parts; ++p) best = merge_best(best, keys[64 * p + 63 - lane], lane);
    }
    write_row<TOP>(a, row, r, best, lane);
}

// Few long rows take workgroups of 1024 threads, whose tile (32768 elements) is
// a whole row of most vocabularies: one launch, no parts.  That is up to a
// workgroup a CU without top tokens, two with (the search for them waits more).
// 32000 logits, 256 / 400 rows without: 6.5 / 12.2 us against 7.5 / 11.1 with 256
// threads; with 20 top tokens 1 / 512 / 768 rows: 8.6 / 22.8 / 32.4 against 17.5 / 25.0 / 29.4.
// The wide forms take 73 registers with top tokens (one workgroup a CU, where 64
// would let in two) and 128 with 11 spilled without.
bool lp_wide(size_t n, size_t rows, size_t k) { return n > 256 * kPer && rows <= (k ? 512 : 256); }
size_t lp_parts(size_t n, size_t rows, size_t k) {
    if (!lp_wide(n, rows, k) || n <= 2 * 1024 * kPer) return 1;
    return std::max<size_t>(1, std::min({(n + 1024 * kPer - 1) / (1024 * kPer), 512 / rows, size_t{64}}));
}

}  // namespace

size_t logprobs_scratch(size_t n, size_t rows, size_t k) {
    const size_t parts = lp_parts(n, rows, k);
    return parts > 1 ? rows * parts * (16 + (k ? 64 * sizeof(u64) : 0)) : 0;
}

hipError_t launch_logprobs(const float* logits, size_t pitch, size_t n, size_t rows, const int* targets, size_t k,
                           float* logprob, float* entropy, int* top_ids, float* top_lp, void* scratch, hipStream_t st) {
    if (!rows) return hipSuccess;
    if (!n || k > 64 || k > n || (logprob && !targets)) return hipErrorInvalidValue;
    LpArgs a{};
    a.logits = logits;
    a.targets = targets;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_lp = top_lp;
    a.n = n;
    a.pitch = pitch;
    a.k = static_cast<int>(k);
    const size_t parts = lp_parts(n, rows, k);
    const size_t tile = (lp_wide(n, rows, k) ? 1024 : 256) * kPer;
    a.chunk = ((n + parts - 1) / parts + tile - 1) / tile * tile;
    a.parts = static_cast<int>((n + a.chunk - 1) / a.chunk);
    if (a.parts > 1) {
        if (!scratch) return hipErrorInvalidValue;
        a.part_keys = static_cast<u64*>(scratch);
        a.part_sums = reinterpret_cast<float*>(a.part_keys + (k ? 64 * rows * a.parts : 0));
    }
    // rows beyond a grid's y range in launches of their own
    for (size_t r0 = 0; r0 < rows; r0 += 65535) {
        const unsigned nr = static_cast<unsigned>(std::min<size_t>(rows - r0, 65535));
        LpArgs b = a;
        b.logits += r0 * pitch;
        if (b.targets) b.targets += r0;
        if (b.logprob) b.logprob += r0;
        if (b.entropy) b.entropy += r0;
        if (b.top_ids) b.top_ids += r0 * k;
        if (b.top_lp) b.top_lp += r0 * k;
        const dim3 grid(static_cast<unsigned>(b.parts), nr);
        if (lp_wide(n, rows, k)) {
            if (k) logprobs_kernel<1024, true><<<grid, 1024, 0, st>>>(b);
            else logprobs_kernel<1024, false><<<grid, 1024, 0, st>>>(b);
        } else {
            if (k) logprobs_kernel<256, true><<<grid, 256, 0, st>>>(b);
            else logprobs_kernel<256, false><<<grid, 256, 0, st>>>(b);
        }
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        if (b.parts > 1) {
            if (k) logprobs_join_kernel<true><<<nr, 64, 0, st>>>(b);
            else logprobs_join_kernel<false><<<nr, 64, 0, st>>>(b);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace mvh
