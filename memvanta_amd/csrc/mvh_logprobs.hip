// mvh_logprobs.hip -- log probabilities of a row of logits: of a given token,
// the entropy, and the most probable tokens.
//
// One pass over the row with a running maximum m:
//   s = sum e^(l - m), t = sum (l - m) e^(l - m),
//   log p_i = (l_i - m) - ln s,  entropy = ln s - t / s,
// all in fp32 per thread, joined across threads with the usual rescaling.  The
// pass is bound by reading the logits (~10 operations an element); few rows are
// cut into parts, whose sums and candidates a second kernel joins.
//
// The most probable tokens: a wave keeps the best 64 keys (value, then lower
// index) sorted across its lanes, and sets aside elements that beat the k-th;
// once 64 wait they are sorted and merged in.  A row of n random elements sets
// aside about k ln(n / k) of them, a sorted one all.
#include "mvh_kernels.hpp"

namespace mvh {
namespace {

constexpr int kLT = 256, kLW = kLT / 64;
constexpr int kPer = 16;               // elements a lane holds at once
constexpr int kBatch = kLT * kPer;     // a workgroup's elements at once
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFar = -1.0e4f;        // e^kFar is 0; keeps 0 * (l - m) from being 0 * inf

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
__device__ __forceinline__ Sums wave_join(Sums a) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) a = join(a, Sums{__shfl_xor(a.m, x), __shfl_xor(a.s, x), __shfl_xor(a.t, x)});
    return a;
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

__device__ __forceinline__ u64 key_xor(u64 k, int x) {
    return (static_cast<u64>(static_cast<uint32_t>(__shfl_xor(static_cast<int>(k >> 32), x))) << 32) |
           static_cast<uint32_t>(__shfl_xor(static_cast<int>(k), x));
}
__device__ __forceinline__ u64 key_at(u64 k, int lane) {
    return (static_cast<u64>(static_cast<uint32_t>(__shfl(static_cast<int>(k >> 32), lane))) << 32) |
           static_cast<uint32_t>(__shfl(static_cast<int>(k), lane));
}
// 64 keys, one a lane, sorted ascending (lane 0 the smallest)
__device__ __forceinline__ u64 sort_ascending(u64 k, int lane) {
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1) {
#pragma unroll
        for (int x = size / 2; x >= 1; x >>= 1) {
            const u64 o = key_xor(k, x);
            const bool up = !(lane & size), first = !(lane & x);
            k = (first == up) == (o < k) ? o : k;
        }
    }
    return k;
}
// best (descending) and more (ascending): the best 64 of both, descending
__device__ __forceinline__ u64 merge_best(u64 best, u64 more, int lane) {
    u64 k = best > more ? best : more;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) {
        const u64 o = key_xor(k, x);
        k = !(lane & x) == (o > k) ? o : k;
    }
    return k;
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

// What the row's results are, from its sums (in every lane of the first wave) and its best keys
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
            if (a.top_ids) a.top_ids[at] = key_index(best);
            if (a.top_lp) a.top_lp[at] = empty ? -INFINITY : (key_value(best) - r.m) - ln_s;
        }
    }
}

template <bool TOP>
__global__ __launch_bounds__(kLT) void logprobs_kernel(LpArgs a) {
    __shared__ u64 s_buf[TOP ? kLW : 1][128];
    __shared__ Sums s_sums[kLW];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const size_t row = blockIdx.y, begin = blockIdx.x * a.chunk, end = min(begin + a.chunk, a.n);
    const float* x = a.logits + row * a.pitch;
    Sums r = {-3.402823466e38f, 0.0f, 0.0f};
    Best top;
    top.buf = s_buf[TOP ? wave : 0];
    top.lane = lane;
    top.k = a.k;
    float v[kPer], w[kPer];
    // batch b of this wave: four times 256 consecutive elements, four a lane
    auto load = [&](size_t at, float (&d)[kPer]) {
#pragma unroll
        for (int c = 0; c < kPer / 4; ++c) {
            const size_t i = at + c * 256 + lane * 4;
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
    size_t at = begin + static_cast<size_t>(wave) * (kBatch / kLW);
    if (at < end) load(at, v);
    bool first = true;
    for (; at < end; at += kBatch) {
        if (at + kBatch < end) load(at + kBatch, w);
        float bm = v[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) bm = fmaxf(bm, v[i]);
        const float m = fmaxf(r.m, bm), dm = fmaxf(r.m - m, kFar), f = __builtin_amdgcn_exp2f(dm * kLog2e);
        float s = r.s * f, t = f * fmaf(dm, r.s, r.t);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float d = v[i] - m, p = __builtin_amdgcn_exp2f(d * kLog2e);
            s += p;
            t = fmaf(p, fmaxf(d, kFar), t);
        }
        r = {m, s, t};
        if constexpr (TOP) {
            if (first) {
                // the k-th largest of the lanes' largest is at most the k-th best of the batch
                u64 mine = 0;
#pragma unroll
                for (int c = 0; c < kPer; ++c) {
                    const size_t i = at + (c / 4) * 256 + lane * 4 + c % 4;
                    const u64 key = i < end ? key_of(v[c], static_cast<int>(i)) : 0;
                    mine = key > mine ? key : mine;
                }
                const u64 floor_key = key_at(sort_ascending(mine, lane), 64 - a.k);
                top.least = floor_key ? floor_key - 1 : 0;
            }
            // equal values of later batches have higher indices: they lose
            if (first || top.least == 0 || __any(bm > key_value(top.least))) {
#pragma unroll
                for (int c = 0; c < kPer; ++c) {
                    const size_t i = at + (c / 4) * 256 + lane * 4 + c % 4;
                    top.offer(i < end ? key_of(v[c], static_cast<int>(i)) : 0);
                }
            }
            first = false;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = w[i];
    }
    if constexpr (TOP) {
        while (top.waiting > 0) top.flush();
        __syncthreads();
        s_buf[wave][lane] = top.best;
    }
    r = wave_join(r);
    if (lane == 0) s_sums[wave] = r;
    __syncthreads();
    if (wave) return;
    u64 best = top.best;
    for (int k = 1; k < kLW; ++k) {
        r = join(r, s_sums[k]);
        if constexpr (TOP) best = merge_best(best, s_buf[k][63 - lane], lane);
    }
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
    r = wave_join(r);
    u64 best = 0;
    if constexpr (TOP) {
        const u64* keys = a.part_keys + 64 * row * a.parts;
        best = keys[lane];
        for (int p = 1; p < a.parts; ++p) best = merge_best(best, keys[64 * p + 63 - lane], lane);
    }
    write_row<TOP>(a, row, r, best, lane);
}

// Parts of a row: about two workgroups a CU over all rows, each at least one batch
size_t lp_parts(size_t n, size_t rows) {
    const size_t most = (n + kBatch - 1) / kBatch;
    return std::max<size_t>(1, std::min({most, 512 / rows, size_t{64}}));
}

}  // namespace

size_t logprobs_scratch(size_t n, size_t rows, size_t k) {
    const size_t parts = lp_parts(n, rows);
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
    const size_t parts = lp_parts(n, rows);
    a.chunk = ((n + parts - 1) / parts + kBatch - 1) / kBatch * kBatch;
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
        if (k) logprobs_kernel<true><<<grid, kLT, 0, st>>>(b);
        else logprobs_kernel<false><<<grid, kLT, 0, st>>>(b);
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
