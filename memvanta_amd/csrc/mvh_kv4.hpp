// mvh_kv4.hpp -- layout of a KV cache page held in 4 bits (kKvQ4).
//
// A row of kv_dim elements is cut into blocks of 32.  A block stands for
//   x = c + s (n - 8),  n in 0..15,
// with s = fp16((max - min) / 15) (at most 512), c = fp16(min + 8 s) and
// n = round((x - c) / s) + 8: 5 bits an element.  A block with a NaN or an
// infinity in it has s = NaN, c = 0 and reads as NaN; c is always finite.
//
// The page is laid out for the matrix pipe, which takes operands of 8
// consecutive contraction elements per lane: rows (slots) in groups of 8, and
// per block and group 32 words of 8 nibbles,
//   K: a word holds 8 consecutive channels (8 kq ..) of one row; row i + 4 u
//      at word (kq * 4 + i) * 2 + u, so that one 8-byte load gives a lane the
//      two rows (u = 0, 1) of its two 16-row tiles;
//   V: a word holds the 8 rows of one channel; channel c + 16 h at word c * 2
//      + h, so that one 8-byte load gives a lane its two 16-channel tiles.
// The page is [block][group] of these 128 bytes, then [block][group] of the
// rows' scales: dwords of s for rows (0, 4), (1, 5), (2, 6), (7, 3), then four
// dwords of c in the same order.  Consecutive rows of a block are consecutive
// in memory.
//
// A word is stored rotated left by 6, which puts nibbles 0 and 4 where the
// upper four mantissa bits of two fp16 are, and 7 and 3 four bits below: with
// the word rotated by 8 once, four and-ors and packed subtractions unpack all
// eight (q4_unpack), in the order of the scales.
#pragma once
#include "mvh_device.hpp"

namespace mvh {

constexpr int kQ4Block = 32;
constexpr float kQ4MaxStep = 512.0f;  // keeps 64 p s within fp16 in the attention kernels

__host__ __device__ constexpr size_t kv4_groups(size_t page_tokens) { return (page_tokens + 7) / 8; }
__host__ __device__ constexpr size_t kv4_scales(size_t page_tokens, size_t kv_dim) {  // offset of the scales
    return kv_dim / 32 * kv4_groups(page_tokens) * 128;
}
// word index within a group's 128 bytes
__host__ __device__ constexpr int kv4_k_word(int row, int kq) { return (kq * 4 + (row & 3)) * 2 + (row >> 2); }
__host__ __device__ constexpr int kv4_v_word(int ch) { return (ch & 15) * 2 + (ch >> 4); }

// natural word (nibble j at bits 4j..) <-> stored word
__host__ __device__ constexpr uint32_t kv4_store(uint32_t nat) { return (nat << 6) | (nat >> 26); }
__host__ __device__ constexpr uint32_t kv4_nat(uint32_t w) { return (w >> 6) | (w << 26); }

// The 8 values n - 8 of a stored word as fp16 (exact), in the order of
// nibbles 0 4 1 5 2 6 7 3: 0x4c00 | n << 6 is 16 + n, 0x5c00 | n << 2 is 256 + n.
// The or's constants come in registers (an instruction takes one literal).
struct Q4Ones {
    uint32_t c16 = 0x4c004c00u, c256 = 0x5c005c00u;
};
__device__ __forceinline__ half8 q4_unpack(uint32_t w, const Q4Ones& k) {
    const uint32_t r = __builtin_amdgcn_alignbit(w, w, 8);
    const _Float16 m24 = static_cast<_Float16>(-24.0f), m264 = static_cast<_Float16>(-264.0f);
    const u32x4 v = {as_u32(as_half2((w & 0x03c003c0u) | k.c16) + m24), as_u32(as_half2((r & 0x003c003cu) | k.c256) + m264),
                     as_u32(as_half2((r & 0x03c003c0u) | k.c16) + m24), as_u32(as_half2((w & 0x003c003cu) | k.c256) + m264)};
    return __builtin_bit_cast(half8, v);
}

// Index of row `row` (0..7) of a group among its 8 steps (or middles)
__host__ __device__ constexpr int kv4_scale(int row) { return (row & 3) * 2 + ((row >> 2) ^ ((row & 3) == 3 ? 1 : 0)); }
// Step and middle of a row: base = the group's 32 bytes of scales
__device__ __forceinline__ float kv4_step(const uint8_t* base, int row) {
    return h2f(reinterpret_cast<const uint16_t*>(base)[kv4_scale(row)]);
}
__device__ __forceinline__ float kv4_middle(const uint8_t* base, int row) {
    return h2f(reinterpret_cast<const uint16_t*>(base)[8 + kv4_scale(row)]);
}

// Row order with each page's rows rounded up to whole groups: group index of a
// position, and back.  page_of divides by the groups per page through a 2^40
// reciprocal, exact for indexes below 2^21 and up to 2^17 groups a page.
struct Kv4Map {
    int page_tokens = 0, groups = 0;
    uint64_t recip = 0;  // floor(2^40 / groups) + 1
    __host__ __device__ int group_of(int pos) const {
        return pos / page_tokens * groups + pos % page_tokens / 8;
    }
    __device__ __forceinline__ int page_of(int vg) const {
        return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(vg)) * recip) >> 40);
    }
};
inline Kv4Map kv4_map(size_t page_tokens) {
    Kv4Map m;
    m.page_tokens = static_cast<int>(page_tokens);
    m.groups = static_cast<int>(kv4_groups(page_tokens));
    m.recip = (uint64_t{1} << 40) / static_cast<uint64_t>(m.groups) + 1;
    return m;
}

}  // namespace mvh
