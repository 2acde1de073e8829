// What the operators on 8-bit floating point rows share (e4m3: one sign, four exponent and three fraction bits, largest value 448, a NaN, no infinity).
//
// Rows are held as q[row][channel] with one fp32 scale for 128 channels of a row (weights: of 128 rows): value = q * scale,
//   scale = max(max|y| / 448, 2^-126),  q = e4m3(y / scale), to nearest, ties to even.
// The smallest scale is a normal number, so that a block of zeros needs no case of its own and a quotient is never above 448 (1 + 2^-23), which rounds to 448.
// The maximum passes over NaN: one stays where it is.  An infinity makes its block's scale infinite and all of its values NaN.
#pragma once

#include "kv_common.hpp"

namespace onhip {

constexpr int F8_BLOCK = 128;

// the type names of the C interface (ONHIP_COMPUTE_*) as element types of rows
inline bool element_type(int compute, int *dt) {
    *dt = compute == ONHIP_COMPUTE_F32 ? DT_F32 : compute == ONHIP_COMPUTE_BF16 ? DT_BF16 : DT_F16;
    return compute == ONHIP_COMPUTE_F32 || compute == ONHIP_COMPUTE_BF16 || compute == ONHIP_COMPUTE_F16;
}
template <int DT> constexpr int element_bytes = DT == DT_F32 ? 4 : 2;
inline int bytes_of(int dt) { return dt == DT_F32 ? 4 : 2; }

template <int DT> __device__ __forceinline__ float widened(unsigned short x) {
    if constexpr (DT == DT_BF16) return __uint_as_float((unsigned) x << 16);
    else return (float) __builtin_bit_cast(_Float16, x);
}

// sixteen bytes at an element's alignment: global memory takes them in one access wherever they lie, at an aligned place as fast as any (1463 fp32 rows of 12135 channels, which start
// everywhere, through the norm: 51 us, 132 with an element an access)
typedef unsigned any_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned any_u32x2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float any_f32x4 __attribute__((ext_vector_type(4), aligned(4)));

// eight consecutive elements at `at`, of which `left` exist (the others are zeros)
template <int DT> __device__ __forceinline__ void load8(const char *at, int left, float (&v)[8]) {
    if (left >= 8) {
        if constexpr (DT == DT_F32) {
            const any_f32x4 a = reinterpret_cast<const any_f32x4 *>(at)[0], b = reinterpret_cast<const any_f32x4 *>(at)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const any_u32x4 w = *reinterpret_cast<const any_u32x4 *>(at);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = widened<DT>((unsigned short) w[j]);
                v[2 * j + 1] = widened<DT>((unsigned short) (w[j] >> 16));
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = 0.0f;
        if (j < left) {
            if constexpr (DT == DT_F32) v[j] = reinterpret_cast<const float *>(at)[j];
            else v[j] = widened<DT>(reinterpret_cast<const unsigned short *>(at)[j]);
        }
    }
}

template <int DT> __device__ __forceinline__ void store8(char *at, int left, const float (&v)[8]) {
    unsigned w[4];
    if constexpr (DT != DT_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_h16<DT>(v[2 * j], v[2 * j + 1]);
    }
    if (left >= 8) {
        if constexpr (DT == DT_F32) {
            reinterpret_cast<any_f32x4 *>(at)[0] = any_f32x4{v[0], v[1], v[2], v[3]};
            reinterpret_cast<any_f32x4 *>(at)[1] = any_f32x4{v[4], v[5], v[6], v[7]};
        } else {
            *reinterpret_cast<any_u32x4 *>(at) = any_u32x4{w[0], w[1], w[2], w[3]};
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) {
            if constexpr (DT == DT_F32) reinterpret_cast<float *>(at)[j] = v[j];
            else reinterpret_cast<unsigned short *>(at)[j] = (unsigned short) (w[j / 2] >> (j % 2 * 16));
        }
}

// the largest magnitude of a block whose values sixteen lanes have, eight each; NaN is passed over, and a block of nothing else has 0
__device__ __forceinline__ float block_top(const float (&y)[8]) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(y[j]));
    top = fmaxf(top, lane_moved<DPP_XOR1>(top));
    top = fmaxf(top, lane_moved<DPP_XOR2>(top));
    top = fmaxf(top, lane_moved<DPP_MIRROR8>(top));
    return fmaxf(top, lane_moved<DPP_MIRROR16>(top));
}

// top / 448, rounded correctly (one step of the division's remainder behind the product with the reciprocal), 2^-126 at least
__device__ __forceinline__ float f8_scale(float top) {
    constexpr float R = 1.0f / 448.0f;
    const float q = top * R, r = __builtin_fmaf(-q, 448.0f, top);
    const float s = __builtin_fmaf(r, R, q);
    return top < INFINITY ? fmaxf(s, 0x1p-126f) : top;
}

// y / scale as eight e4m3.  The quotient is the product with the reciprocal and one step of the remainder: as the division rounds it, so that a value in the
// middle of two e4m3 goes to the even one
__device__ __forceinline__ uint2 f8_pack(const float (&y)[8], float scale) {
    float inv = __builtin_amdgcn_rcpf(scale);
    inv = __builtin_fmaf(__builtin_fmaf(-scale, inv, 1.0f), inv, inv);
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = y[j] * inv;
        z[j] = __builtin_fmaf(-__builtin_fmaf(q, scale, -y[j]), inv, q);   // signs so that -0 stays -0
    }
    uint2 o;
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false), b = __builtin_amdgcn_cvt_pk_fp8_f32(z[4], z[5], 0, false);
    o.x = (unsigned) __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], a, true);
    o.y = (unsigned) __builtin_amdgcn_cvt_pk_fp8_f32(z[6], z[7], b, true);
    return o;
}

// eight bytes of a row; rows are 16-byte aligned
__device__ __forceinline__ void f8_store(char *at, int left, uint2 q) {
    if (left >= 8) {
        *reinterpret_cast<uint2 *>(at) = q;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) at[j] = (char) ((j < 4 ? q.x : q.y) >> (j % 4 * 8));
}

// workgroups in rows of 2^21, for a row's threads are counted in 32 bits; what is behind the last one returns
inline dim3 f8_grid(long long groups) { return dim3((unsigned) (groups < (1 << 21) ? groups : 1 << 21), (unsigned) ((groups + (1 << 21) - 1) >> 21)); }
__device__ __forceinline__ long long f8_group() { return (long long) blockIdx.y * (1 << 21) + blockIdx.x; }

inline bool misaligned(const void *at, uintptr_t to) { return reinterpret_cast<uintptr_t>(at) % to != 0; }

// rows of bytes as a call names them, and whether two of them have no byte in common: spans behind each other, or columns of one matrix
struct Span {
    const char *at;
    long long step, row;   // bytes
    int rows;
};
inline bool apart(const Span &a, const Span &b) {
    if (!a.at || !b.at) return true;
    auto last = [](const Span &x) { return x.at + (x.rows - 1) * x.step + x.row; };
    if (last(a) <= b.at || last(b) <= a.at) return true;
    const long long step = a.rows > 1 ? a.step : b.step;
    if ((a.rows > 1 && b.rows > 1 && a.step != b.step) || step == 0) return false;
    long long off = (b.at - a.at) % step;
    off = off < 0 ? off + step : off;
    return off >= a.row && off + b.row <= step;
}
// scales as one span of bytes
inline Span scale_span(const float *scale, const long long *ss, int rows, int blocks) {
    return {reinterpret_cast<const char *>(scale), 0, 4 * ((rows - 1) * ss[0] + (blocks - 1) * ss[1] + 1), 1};
}
inline bool same(const Span &a, const Span &b) { return a.at == b.at && a.step == b.step && a.row == b.row; }

}  // namespace onhip
