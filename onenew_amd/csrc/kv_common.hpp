// What the kernels on a paged key-value cache share: where a token's row lies, and the checks of a cache's description.
#pragma once

#include "igemm_kernel.hpp"

namespace onhip {

// The cache as kernels see it: strides of (page, head, row) in bytes for k and v, in floats for the scales.
struct CacheView {
    char *k, *v;
    float *k_scale, *v_scale;
    long long ks[3], vs[3], ss[3];
    int pages, page_shift, page_mask;
};

// checks the description and fills the view's sizes and strides; `what` names the entry point in the message
int cache_shape(const char *what, const onhip_cache_desc_t *c, CacheView *view, int *dt);
// checks the addresses and fills them in
int cache_memory(const char *what, const onhip_cache_desc_t *c, const void *k, const void *v, const float *k_scale, const float *v_scale, CacheView *view);

// Whether every row of `row` elements has memory of its own under these extents and strides (in elements, not negative; an extent of one has none):
// each stride is at least the span of the extents with smaller ones.  Rows that share memory would be written by several wavefronts.
template <int N> inline bool rows_apart(const int (&extent)[N], const long long *stride, long long row) {
    int order[N];
    for (int i = 0; i < N; ++i) {
        int at = i;
        for (; at > 0 && stride[order[at - 1]] > stride[i]; --at) order[at] = order[at - 1];
        order[at] = i;
    }
    __int128 span = row;
    for (int i : order) {
        if (extent[i] <= 1) continue;
        if (stride[i] < span) return false;
        span += (__int128) stride[i] * (extent[i] - 1);
    }
    return true;
}

// lane i's value from lane i ^ 1, i ^ 2, 7 - i (of eight) or 15 - i (of sixteen), through the vector pipe
enum { DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_REVERSE4 = 0x1B, DPP_MIRROR8 = 0x141, DPP_MIRROR16 = 0x140, DPP_ROTATE8 = 0x128 };
template <int HOW> __device__ __forceinline__ unsigned lane_moved(unsigned x) { return (unsigned) __builtin_amdgcn_update_dpp(0, (int) x, HOW, 0xf, 0xf, true); }
template <int HOW> __device__ __forceinline__ float lane_moved(float x) { return __uint_as_float(lane_moved<HOW>(__float_as_uint(x))); }

// eight signed bytes as pairs of the 16-bit type: every int8 is a bf16 and an fp16
template <int DT> __device__ __forceinline__ void s8_to_h16(const unsigned (&x)[2], unsigned (&y)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int w = (int) x[i];
        y[2 * i] = pack_h16<DT>((float) (signed char) w, (float) (signed char) (w >> 8));
        y[2 * i + 1] = pack_h16<DT>((float) (signed char) (w >> 16), (float) (signed char) (w >> 24));
    }
}

}  // namespace onhip
