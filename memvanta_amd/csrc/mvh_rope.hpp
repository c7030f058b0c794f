// mvh_rope.hpp -- rotation of a head's elements by its token's position.
//
// A pair (x0, x1) of the rotated part turns by the angle pos * f_i: y0 = x0 c
// - x1 s, y1 = x0 s + x1 c.  Angles of far positions need more than 32 bits
// (pos * f_i reaches 1e5 and more, where fp32 steps by 0.01), so the angle,
// its reduction, sine and cosine are taken in double and rounded once; the
// products and the sum are fp32, each rounded.
#pragma once
#include "mvh_device.hpp"

namespace mvh {

enum RopeLayout : int { kRopeHalf = 0, kRopeInterleaved = 1 };

// What a rotation needs on the device: freq[i] = angle per position of pair i
// (rot / 2 doubles), in device memory.
struct RopeView {
    const double* freq = nullptr;
    double scale = 1.0;  // of the rotated part
    int head_dim = 0, rot = 0, layout = kRopeHalf;
};

// sin and cos of an angle: the nearest multiple k of pi/2 taken off with pi/2
// in two doubles (k < 2^51, of 2^31 positions and factors of 2^-20: the fused
// products keep the rest exact to 1e-16), then the Taylor series on |y| <= pi/4,
// cut where the next term is below 2^-45 -- 2^-21 of half an fp32 step (1.1,
// where k from 2^49 on is off by one: 2^-38).
__device__ __forceinline__ void sin_cos(double a, double& s, double& c) {
    const double k = rint(a * 0.63661977236758134308);
    double y = fma(-k, 1.57079632679489655800, a);
    y = fma(-k, 6.12323399573676603587e-17, y);
    const double z = y * y;
    double p = 1.0 / 6227020800.0;
    p = fma(p, z, -1.0 / 39916800.0);
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, -1.0 / 5040.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, -1.0 / 6.0);
    const double sy = fma(p * z, y, y);
    double q = -1.0 / 87178291200.0;
    q = fma(q, z, 1.0 / 479001600.0);
    q = fma(q, z, -1.0 / 3628800.0);
    q = fma(q, z, 1.0 / 40320.0);
    q = fma(q, z, -1.0 / 720.0);
    q = fma(q, z, 1.0 / 24.0);
    q = fma(q, z, -0.5);
    const double cy = fma(q, z, 1.0);
    const int quarter = static_cast<int>(static_cast<long long>(k)) & 3;
    const double u = quarter & 1 ? cy : sy, w = quarter & 1 ? sy : cy;
    s = quarter & 2 ? -u : u;
    c = (quarter + 1) & 2 ? -w : w;
}

// cos (x) and sin (y) of pair i at position pos, times the scale
__device__ __forceinline__ float2 rope_turn(const RopeView& r, int pos, int i) {
    double s, c;
    sin_cos(static_cast<double>(pos) * r.freq[i], s, c);
    return make_float2(static_cast<float>(r.scale * c), static_cast<float>(r.scale * s));
}

// Elements d .. d+3 of one head (x = the head's first element) after the
// rotation; cs = the token's turns.  vec: x 16-byte aligned and a quad's pairs
// lie in one aligned quad (the same, or the one at +-rot/2).
__device__ __forceinline__ float4 rope_quad(const RopeView& r, const float* x, int d, const float2* cs, bool vec) {
    const int half = r.rot / 2;
    float v[4], o[4];
    if (vec) {
        const float4 a = *reinterpret_cast<const float4*>(x + d);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        if (d >= r.rot) return a;
        float w[4];
        int i[4];
        float sgn[4];
        if (r.layout == kRopeHalf) {
            const bool low = d < half;
            const float4 b = *reinterpret_cast<const float4*>(x + (low ? d + half : d - half));
            w[0] = b.x, w[1] = b.y, w[2] = b.z, w[3] = b.w;
#pragma unroll
            for (int j = 0; j < 4; ++j) i[j] = (low ? d : d - half) + j, sgn[j] = low ? -1.0f : 1.0f;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = v[j ^ 1], i[j] = (d + j) / 2, sgn[j] = j & 1 ? 1.0f : -1.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = cs[i[j]];
            o[j] = v[j] * t.x + sgn[j] * (w[j] * t.y);
        }
        return make_float4(o[0], o[1], o[2], o[3]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = d + j;
        if (e >= r.rot) {
            o[j] = x[e];
            continue;
        }
        const bool hf = r.layout == kRopeHalf, low = hf ? e < half : !(e & 1);
        const int i = hf ? (low ? e : e - half) : e / 2, mate = hf ? (low ? e + half : e - half) : e ^ 1;
        const float2 t = cs[i];
        const float a = x[e] * t.x, b = x[mate] * t.y;
        o[j] = low ? a - b : a + b;
    }
    return make_float4(o[0], o[1], o[2], o[3]);
}

}  // namespace mvh
