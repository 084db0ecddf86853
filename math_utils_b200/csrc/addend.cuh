// What a sublayer adds to the float32 stream, shared by the norms that make the addition (qkv_rows.cu, q8_rows.cu).
#pragma once
#include "common.cuh"

namespace mu {

// What a sublayer adds to the stream: (mult * y [+ mult2 * y2]) [* scale, entry by entry].
struct Addend {
    const float* y;           // [rows][ldy], or null: nothing is added
    long long ldy;
    float mult;
    const float* y2;          // a second branch, or null
    long long ldy2;
    float mult2;
    const float* scale;       // [width] or null
};

__device__ __forceinline__ float ra_added(float x, const Addend& a, long long t, long long d) {
    const float y = a.y[t * a.ldy + d];
    if (!a.y2 && !a.scale) return fmaf(a.mult, y, x);
    const float v = a.y2 ? fmaf(a.mult, y, a.mult2 * a.y2[t * a.ldy2 + d]) : a.mult * y;
    return a.scale ? fmaf(v, a.scale[d], x) : x + v;
}
__device__ __forceinline__ float4 ra_added4(float4 x, const Addend& a, long long t, long long d) {
    const float4 y = *reinterpret_cast<const float4*>(a.y + t * a.ldy + d);
    float4 v = make_float4(a.mult * y.x, a.mult * y.y, a.mult * y.z, a.mult * y.w);
    if (a.y2) {
        const float4 u = *reinterpret_cast<const float4*>(a.y2 + t * a.ldy2 + d);
        v = make_float4(fmaf(a.mult2, u.x, v.x), fmaf(a.mult2, u.y, v.y), fmaf(a.mult2, u.z, v.z), fmaf(a.mult2, u.w, v.w));
    }
    if (a.scale) {
        const float4 g = *reinterpret_cast<const float4*>(a.scale + d);
        return make_float4(fmaf(v.x, g.x, x.x), fmaf(v.y, g.y, x.y), fmaf(v.z, g.z, x.z), fmaf(v.w, g.w, x.w));
    }
    return make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
}

}  // namespace mu
