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

// eight (NV = 2) or four (NV = 1) signed bytes as pairs of the 16-bit type: every int8 is a bf16 and an fp16
template <int DT, int NV> __device__ __forceinline__ void s8_to_h16(const unsigned (&x)[NV], unsigned (&y)[2 * NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int w = (int) x[i];
        y[2 * i] = pack_h16<DT>((float) (signed char) w, (float) (signed char) (w >> 8));
        y[2 * i + 1] = pack_h16<DT>((float) (signed char) (w >> 16), (float) (signed char) (w >> 24));
    }
}

}  // namespace onhip
