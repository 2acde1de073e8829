// The paged key-value cache: rows of k and v written into it behind the norm and the position rotation of their heads, and read
// back in sequence order.
//
// Append, for a row x of D values in fp32: x rsqrt(mean(x^2) + eps) w (q and k, where there is a weight), then the first 2 R values
// turned in pairs (a, b) -> (a cos - b sin, b cos + a sin) by the angle position * inv_freq[i]; q goes to its result, k and v to
// the cache at the token's slot, in the 16-bit type or as rint(x 127 / max|x|) in eight bits with the scale max|x| / 127.
//
// A lane has 8 consecutive values of a row (16 bytes in, 16 or 8 out), D / 8 lanes a row, a wavefront four or eight heads of one
// token at a time.  The angles are the token's alone: a lane forms one, the product and its reduction to a revolution in 64 bits
// (position 10^6 times a frequency of 1 keeps 2^-31 of a revolution), and the lanes fetch the cosines of their values from each other.  Sums, maxima and
// the partner values of a full rotation go from lane to lane in the vector pipe (through LDS they and the whole numbers' conversions were
// 49.9 us of the int8 case below).
//
// Bound by memory, and by the vector pipe next to it: 8191 tokens of 32 + 8 + 8 heads of 128 in bf16 201 MB in 41 us with norms and a full rotation, 38 without
// norms (a large copy of as many bytes 40); into an int8 cache 184 MB in 44 (37 of them repeated over one input, part of which the last-level cache holds); a step of 32 tokens 3.3 us, a launch.  Read back: 8 sequences of up to 8192, 8 heads of 128,
// 377 MB of int8 and its values in 75 us, 480 MB of bf16 in 93.
#include "kv_common.hpp"

namespace onhip {

int cache_shape(const char *what, const onhip_cache_desc_t *c, CacheView *view, int *dt) {
    if (!c) return set_error(ONHIP_ERR_ARG, "%s: null cache description", what);
    if (c->compute == ONHIP_COMPUTE_BF16) *dt = DT_BF16;
    else if (c->compute == ONHIP_COMPUTE_F16) *dt = DT_F16;
    else return set_error(ONHIP_ERR_ARG, "%s: compute type %d is neither bf16 nor fp16", what, c->compute);
    if (c->head_dim != 64 && c->head_dim != 128) return set_error(ONHIP_ERR_ARG, "%s: head dimension %d (64 and 128 are available)", what, c->head_dim);
    if (c->pages < 1 || c->kv_heads < 1) return set_error(ONHIP_ERR_ARG, "%s: a cache of %d pages and %d heads", what, c->pages, c->kv_heads);
    if (c->page_tokens < 1 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1)))
        return set_error(ONHIP_ERR_ARG, "%s: pages of %d tokens (a power of two up to 1024)", what, c->page_tokens);
    if ((long long) c->pages * c->page_tokens >= (1LL << 31)) return set_error(ONHIP_ERR_ARG, "%s: a cache of 2^31 tokens or more", what);
    if (c->quantised != 0 && c->quantised != 1) return set_error(ONHIP_ERR_ARG, "%s: quantised = %d", what, c->quantised);
    const int vec = c->quantised ? 16 : 8, extent[3] = {c->pages, c->kv_heads, c->page_tokens};
    const long long *strides[2] = {c->k_strides, c->v_strides};
    for (int t = 0; t < 2; ++t)
        for (int i = 0; i < 3; ++i) {
            if (extent[i] == 1) continue;   // never stepped over
            if (strides[t][i] < c->head_dim || strides[t][i] % vec)
                return set_error(ONHIP_ERR_ARG, "%s: cache strides must be multiples of %d, at least the head dimension", what, vec);
        }
    for (int t = 0; t < 2; ++t)
        if ((c->page_tokens > 1 && strides[t][2] >= (1LL << 30) / c->page_tokens)) return set_error(ONHIP_ERR_ARG, "%s: page tokens x row stride reaches 2^30", what);
    if (c->quantised)
        for (int i = 0; i < 3; ++i)
            if (extent[i] > 1 && (c->scale_strides[i] < 1 || (i == 2 && c->scale_strides[i] >= (1LL << 30) / c->page_tokens)))
                return set_error(ONHIP_ERR_ARG, "%s: bad scale strides", what);
    const int size = c->quantised ? 1 : 2;
    for (int i = 0; i < 3; ++i) {
        view->ks[i] = extent[i] == 1 ? 0 : c->k_strides[i] * size;
        view->vs[i] = extent[i] == 1 ? 0 : c->v_strides[i] * size;
        view->ss[i] = extent[i] == 1 ? 0 : c->scale_strides[i];
    }
    view->pages = c->pages;
    view->page_shift = __builtin_ctz((unsigned) c->page_tokens);
    view->page_mask = c->page_tokens - 1;
    return ONHIP_OK;
}

int cache_memory(const char *what, const onhip_cache_desc_t *c, const void *k, const void *v, const float *k_scale, const float *v_scale, CacheView *view) {
    if (!k || !v) return set_error(ONHIP_ERR_ARG, "%s: null cache pointer", what);
    if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return set_error(ONHIP_ERR_ARG, "%s: the cache must be 16-byte aligned", what);
    if (c->quantised && (!k_scale || !v_scale)) return set_error(ONHIP_ERR_ARG, "%s: an int8 cache needs its scales", what);
    if (c->quantised && (reinterpret_cast<uintptr_t>(k_scale) % 4 || reinterpret_cast<uintptr_t>(v_scale) % 4))
        return set_error(ONHIP_ERR_ARG, "%s: misaligned scales", what);
    view->k = const_cast<char *>(reinterpret_cast<const char *>(k));   // cache_append alone writes through them
    view->v = const_cast<char *>(reinterpret_cast<const char *>(v));
    view->k_scale = const_cast<float *>(k_scale);
    view->v_scale = const_cast<float *>(v_scale);
    return ONHIP_OK;
}

struct AppendParams {
    CacheView c;
    const unsigned short *q, *k, *v;
    unsigned short *q_out;
    long long qs[2], ks[2], vs[2], os[2];   // elements: (token, head)
    const int *positions, *slots;
    const float *inv_freq, *q_weight, *k_weight;
    int tokens, q_heads, kv_heads, pairs;
    float eps;
    int waves;       // wavefronts that share a token's heads
};

// over the LANES lanes of a row: each step joins groups that the last one made equal
template <int LANES> __device__ __forceinline__ unsigned row_max(unsigned x) {
    x = max(x, lane_moved<DPP_XOR1>(x));
    x = max(x, lane_moved<DPP_XOR2>(x));
    x = max(x, lane_moved<DPP_MIRROR8>(x));
    return LANES == 16 ? max(x, lane_moved<DPP_MIRROR16>(x)) : x;
}
template <int LANES> __device__ __forceinline__ float row_sum(float x) {
    x += lane_moved<DPP_XOR1>(x);
    x += lane_moved<DPP_XOR2>(x);
    x += lane_moved<DPP_MIRROR8>(x);
    return LANES == 16 ? x + lane_moved<DPP_MIRROR16>(x) : x;
}
// the value of the lane half a row away
template <int LANES> __device__ __forceinline__ float row_half(float x) {
    return LANES == 16 ? lane_moved<DPP_ROTATE8>(x) : lane_moved<DPP_REVERSE4>(lane_moved<DPP_MIRROR8>(x));
}

// NI: heads that a lane group takes one after the other, all of them asked for before the first is worked on
template <int DT, int HD, bool I8, bool INTERLEAVED, int NI>
__global__ __launch_bounds__(256) void cache_append_kernel(const AppendParams p) {
    constexpr int LANES = HD / 8, GROUPS = 64 / LANES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long item = (long long) blockIdx.x * 4 + wave;
    const int token = (int) (item / p.waves), part = (int) (item - (long long) token * p.waves);
    if (token >= p.tokens) return;   // nothing below synchronises
    const int l = lane % LANES, group = lane / LANES;
    const int heads = p.q_heads + 2 * p.kv_heads;
    const int slot = p.slots[token];
    const bool stored = slot >= 0 && (slot >> p.c.page_shift) < p.c.pages;

    uint4 raw[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int h = (part * NI + i) * GROUPS + group;
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (h < heads) {
            const unsigned short *src = h < p.q_heads ? p.q + token * p.qs[0] + h * p.qs[1]
                                        : h < p.q_heads + p.kv_heads ? p.k + token * p.ks[0] + (h - p.q_heads) * p.ks[1]
                                                                     : p.v + token * p.vs[0] + (h - p.q_heads - p.kv_heads) * p.vs[1];
            raw[i] = *reinterpret_cast<const uint4 *>(src + l * 8);
        }
    }
    // the angle of pair `lane`, as a fraction of a revolution
    float cs = 1.0f, sn = 0.0f;
    if (lane < p.pairs) {
        const double rev = (double) p.positions[token] * ((double) p.inv_freq[lane] * 0.15915494309189533577);
        sincospif(2.0f * (float) (rev - rint(rev)), &sn, &cs);
    }
    // this lane's values: element e of the row belongs to pair e % R (or e / 2) of those below 2 R
    float c8[8], s8[8];
    bool turned = false;
    int partner = lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = l * 8 + j;
        const int pair = INTERLEAVED ? e / 2 : e < p.pairs ? e : e - p.pairs;
        c8[j] = __shfl(cs, pair & 63, 64);
        s8[j] = __shfl(sn, pair & 63, 64);
    }
    if (l * 8 < 2 * p.pairs) {   // pairs is a multiple of 8: all of a lane's values or none
        turned = true;
        if (!INTERLEAVED) {
            const bool first = l * 8 < p.pairs;
            partner = first ? lane + p.pairs / 8 : lane - p.pairs / 8;
            if (first)
#pragma unroll
                for (int j = 0; j < 8; ++j) s8[j] = -s8[j];
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int h = (part * NI + i) * GROUPS + group;
        const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
        float x[8];
        const unsigned w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = unpack_h16<DT>(w[j / 2], j % 2);
        const float *weight = is_q ? p.q_weight : p.k_weight;
        const bool normed = !is_v && weight != nullptr;
        float r = 1.0f;
        if (p.q_weight || p.k_weight) {   // uniform
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
            sum = row_sum<LANES>(sum);
            if (normed) r = rsqrtf(sum * (1.0f / HD) + p.eps);
        }
        if (normed)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * r * weight[l * 8 + j];
        if (p.pairs > 0) {   // uniform
            float y[8];
            if (INTERLEAVED) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    y[j] = __builtin_fmaf(x[j], c8[j], -(x[j + 1] * s8[j]));
                    y[j + 1] = __builtin_fmaf(x[j + 1], c8[j], x[j] * s8[j]);
                }
            } else if (2 * p.pairs == HD) {   // uniform
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = __builtin_fmaf(x[j], c8[j], row_half<LANES>(x[j]) * s8[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = __builtin_fmaf(x[j], c8[j], __shfl(x[j], partner, 64) * s8[j]);
            }
            if (turned && !is_v)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = y[j];
        }
        const uint4 packed = make_uint4(pack_h16<DT>(x[0], x[1]), pack_h16<DT>(x[2], x[3]), pack_h16<DT>(x[4], x[5]), pack_h16<DT>(x[6], x[7]));
        unsigned top_bits = 0u;   // of max|x|: as whole numbers, an infinity is above every number and a NaN above that
        if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) top_bits = max(top_bits, __float_as_uint(x[j]) & 0x7fffffffu);
            top_bits = row_max<LANES>(top_bits);
        }
        if (h >= heads) continue;
        if (is_q) {
            *reinterpret_cast<uint4 *>(p.q_out + token * p.os[0] + h * p.os[1] + l * 8) = packed;
            continue;
        }
        if (!stored) continue;
        const int kh = is_v ? h - p.q_heads - p.kv_heads : h - p.q_heads, page = slot >> p.c.page_shift, row = slot & p.c.page_mask;
        char *dst = is_v ? p.c.v + page * p.c.vs[0] + kh * p.c.vs[1] + row * p.c.vs[2] : p.c.k + page * p.c.ks[0] + kh * p.c.ks[1] + row * p.c.ks[2];
        if constexpr (!I8) {
            *reinterpret_cast<uint4 *>(dst + l * 16) = packed;
        } else {
            const bool fine = top_bits < 0x7f800000u;
            const float top = __uint_as_float(top_bits);
            // 127 / max leaves fp32's range below 2^-121, and the reciprocal its normal numbers above 2^126: such rows are scaled first, exactly
            float up = 1.0f;
            if (__any(top < 0x1p-100f || top > 0x1p100f)) {
                up = top < 0x1p-100f ? 0x1p100f : top > 0x1p100f ? 0x1p-100f : 1.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= up;
            }
            // x 127 / max by the reciprocal, which is a unit off, and one step of the division's remainder: a quotient that fp32 holds comes out as it is, so that one in the
            // middle of two whole numbers goes to the even one (by the reciprocal alone half of the largest value of some rows was 63 and not 64)
            const float size = top * up, inv = top > 0.0f && fine ? __builtin_amdgcn_rcpf(size) : 0.0f;
            // to the nearest whole number by adding 1.5 2^23, whose sum has it in its lowest byte
            unsigned b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[j] * 127.0f, z = y * inv;
                b[j] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-z, size, y), inv, z) + 12582912.0f);
            }
            unsigned q8[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                q8[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * j + 3], b[4 * j + 2], 0x0c0c0400u), __builtin_amdgcn_perm(b[4 * j + 1], b[4 * j], 0x0c0c0400u), 0x05040100u);
            *reinterpret_cast<uint2 *>(dst + l * 8) = fine ? make_uint2(q8[0], q8[1]) : make_uint2(0u, 0u);
            if (l == 0) (is_v ? p.c.v_scale : p.c.k_scale)[page * p.c.ss[0] + kh * p.c.ss[1] + row * p.c.ss[2]] = fine ? top * (1.0f / 127.0f) : NAN;
        }
    }
}

template <int DT, int HD, bool I8, bool INTERLEAVED>
static int append_launch(AppendParams p, hipStream_t stream) {
    const int rounds = (p.q_heads + 2 * p.kv_heads + 512 / HD - 1) / (512 / HD);   // of a wavefront's four or eight heads
    const bool many = (long long) p.tokens * rounds > 8192 && rounds > 1;
    p.waves = many ? (rounds + 3) / 4 : rounds;
    const long long blocks = ((long long) p.tokens * p.waves + 3) / 4;
    if (blocks >= (1LL << 31)) return set_error(ONHIP_ERR_ARG, "cache append: %d tokens of %d heads", p.tokens, p.q_heads + 2 * p.kv_heads);
    if (many) hipLaunchKernelGGL((cache_append_kernel<DT, HD, I8, INTERLEAVED, 4>), dim3((unsigned) blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((cache_append_kernel<DT, HD, I8, INTERLEAVED, 1>), dim3((unsigned) blocks), dim3(256), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

// ---- the cache's rows in sequence order --------------------------------------------------------------------------
struct ReadParams {
    CacheView c;
    unsigned short *k_out, *v_out;
    long long os[2][3];   // elements: (sequence, head, token)
    const int *table, *lengths;
    long long table_stride;
    int table_pages, batch, kv_heads, tokens;
};

// A workgroup copies ROWS rows of one head of one sequence, k or v; a lane 8 values of NR rows, all asked for before the first is stored.
template <int DT, int HD, bool I8>
__global__ __launch_bounds__(256) void cache_read_kernel(const ReadParams p) {
    constexpr int LANES = HD / 8, GROUPS = 256 / LANES, NR = 4;
    const int l = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int b = blockIdx.z >> 1, is_v = blockIdx.z & 1, h = blockIdx.y;
    const int reach = p.lengths[b];
    const char *base = is_v ? p.c.v + h * p.c.vs[1] : p.c.k + h * p.c.ks[1];
    const long long s0 = is_v ? p.c.vs[0] : p.c.ks[0], s2 = is_v ? p.c.vs[2] : p.c.ks[2];
    const float *scales = is_v ? p.c.v_scale : p.c.k_scale;
    const int first = blockIdx.x * (GROUPS * NR) + group;
    int page[NR];
    bool there[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int t = first + i * GROUPS;
        there[i] = t < p.tokens && t < reach;
        page[i] = -1;
        if (there[i] && (t >> p.c.page_shift) < p.table_pages) page[i] = p.table[b * p.table_stride + (t >> p.c.page_shift)];
    }
    unsigned w[NR][4];
    float scale[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int t = first + i * GROUPS, row = t & p.c.page_mask;
        const bool good = there[i] && (unsigned) page[i] < (unsigned) p.c.pages;
        w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0u;
        scale[i] = there[i] ? NAN : 0.0f;   // rows behind the last token are zeros, rows on a page that does not exist NaN
        if (good) {
            const char *src = base + page[i] * s0 + row * s2;
            if constexpr (I8) {
                const uint2 x = *reinterpret_cast<const uint2 *>(src + l * 8);
                w[i][0] = x.x; w[i][1] = x.y;
                scale[i] = scales[page[i] * p.c.ss[0] + h * p.c.ss[1] + row * p.c.ss[2]];
            } else {
                const uint4 x = *reinterpret_cast<const uint4 *>(src + l * 16);
                w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
                scale[i] = 0.0f;
            }
        }
    }
    unsigned short *out = (is_v ? p.v_out : p.k_out) + b * p.os[is_v][0] + h * p.os[is_v][1];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int t = first + i * GROUPS;
        if (t >= p.tokens) continue;
        uint4 y = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
        if constexpr (I8) {
            unsigned o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int x = (int) (w[i][j / 2] >> (j % 2 * 16));
                o[j] = pack_h16<DT>((float) (signed char) x * scale[i], (float) (signed char) (x >> 8) * scale[i]);
            }
            y = make_uint4(o[0], o[1], o[2], o[3]);
        } else if (scale[i] != scale[i]) {
            const unsigned nan2 = DT == DT_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
            y = make_uint4(nan2, nan2, nan2, nan2);
        }
        *reinterpret_cast<uint4 *>(out + t * p.os[is_v][2] + l * 8) = y;
    }
}

template <int DT, int HD, bool I8>
static int read_launch(const ReadParams &p, hipStream_t stream) {
    constexpr int ROWS = 256 / (HD / 8) * 4;
    const dim3 grid((unsigned) ((p.tokens + ROWS - 1) / ROWS), (unsigned) p.kv_heads, (unsigned) p.batch * 2u);
    hipLaunchKernelGGL((cache_read_kernel<DT, HD, I8>), grid, dim3(256), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

}  // namespace onhip

using namespace onhip;

extern "C" {

int onhip_cache_append(const onhip_cache_desc_t *c, void *k_cache, void *v_cache, float *k_scale, float *v_scale,
                       const onhip_cache_rows_desc_t *r, const void *q, const void *k, const void *v, const int32_t *positions,
                       const int32_t *slots, const float *inv_freq, const float *q_weight, const float *k_weight, void *q_out, void *stream) {
    AppendParams p;
    int dt, rc = cache_shape("cache append", c, &p.c, &dt);
    if (!rc) rc = cache_memory("cache append", c, k_cache, v_cache, k_scale, v_scale, &p.c);
    if (rc) return rc;
    if (!r || r->tokens < 1 || r->q_heads < 1) return set_error(ONHIP_ERR_ARG, "cache append: bad shape");
    if (r->q_heads > (1 << 20) || c->kv_heads > (1 << 20)) return set_error(ONHIP_ERR_ARG, "cache append: %d and %d heads", r->q_heads, c->kv_heads);
    if (!q || !k || !v || !q_out || !slots) return set_error(ONHIP_ERR_ARG, "cache append: null tensor pointer");
    if (r->pairs < 0 || r->pairs % 8 || 2 * r->pairs > c->head_dim) return set_error(ONHIP_ERR_ARG, "cache append: %d pairs (a multiple of 8, at most half of the head dimension)", r->pairs);
    if (r->pairs && (!positions || !inv_freq)) return set_error(ONHIP_ERR_ARG, "cache append: a rotation needs positions and frequencies");
    if ((q_weight || k_weight) && !(r->eps >= 0.0f)) return set_error(ONHIP_ERR_ARG, "cache append: eps must not be negative");
    if (q_out == k || q_out == v) return set_error(ONHIP_ERR_ARG, "cache append: the result may be q alone");
    const void *ptrs[4] = {q, k, v, q_out};
    const long long *strides[4] = {r->q_strides, r->k_strides, r->v_strides, r->out_strides};
    long long *const own[4] = {p.qs, p.ks, p.vs, p.os};
    for (int t = 0; t < 4; ++t) {
        if (reinterpret_cast<uintptr_t>(ptrs[t]) % 16) return set_error(ONHIP_ERR_ARG, "cache append: tensors must be 16-byte aligned");
        const int extent[2] = {r->tokens, t == 0 || t == 3 ? r->q_heads : c->kv_heads};
        for (int i = 0; i < 2; ++i) {
            own[t][i] = 0;   // a stride that is never stepped over
            if (extent[i] == 1) continue;
            if (strides[t][i] < 0 || strides[t][i] % 8) return set_error(ONHIP_ERR_ARG, "cache append: strides must be non-negative multiples of 8");
            own[t][i] = strides[t][i];
        }
    }
    if (q_out == q && (p.os[0] != p.qs[0] || p.os[1] != p.qs[1])) return set_error(ONHIP_ERR_ARG, "cache append: a result in q's place has q's strides");
    const int out_extent[2] = {r->tokens, r->q_heads}, extent[3] = {c->pages, c->kv_heads, c->page_tokens};
    if (!rows_apart(out_extent, r->out_strides, c->head_dim)) return set_error(ONHIP_ERR_ARG, "cache append: rows of the result overlap");
    if (!rows_apart(extent, c->k_strides, c->head_dim) || !rows_apart(extent, c->v_strides, c->head_dim)) return set_error(ONHIP_ERR_ARG, "cache append: rows of the cache overlap");
    if (c->quantised && !rows_apart(extent, c->scale_strides, 1)) return set_error(ONHIP_ERR_ARG, "cache append: scales of the cache overlap");
    if (k_cache == v_cache || (c->quantised && k_scale == v_scale) || q_out == k_cache || q_out == v_cache)
        return set_error(ONHIP_ERR_ARG, "cache append: one memory for keys and values, or for the result and the cache");
    p.q = reinterpret_cast<const unsigned short *>(q);
    p.k = reinterpret_cast<const unsigned short *>(k);
    p.v = reinterpret_cast<const unsigned short *>(v);
    p.q_out = reinterpret_cast<unsigned short *>(q_out);
    p.positions = positions;
    p.slots = slots;
    p.inv_freq = inv_freq;
    p.q_weight = q_weight;
    p.k_weight = k_weight;
    p.tokens = r->tokens;
    p.q_heads = r->q_heads;
    p.kv_heads = c->kv_heads;
    p.pairs = r->pairs;
    p.eps = r->eps;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto by_order = [&]<int DT, int HD, bool I8>() {
        return r->interleaved ? append_launch<DT, HD, I8, true>(p, st) : append_launch<DT, HD, I8, false>(p, st);
    };
    auto by_size = [&]<int DT>() {
        if (c->head_dim == 64) return c->quantised ? by_order.template operator()<DT, 64, true>() : by_order.template operator()<DT, 64, false>();
        return c->quantised ? by_order.template operator()<DT, 128, true>() : by_order.template operator()<DT, 128, false>();
    };
    return dt == DT_BF16 ? by_size.template operator()<DT_BF16>() : by_size.template operator()<DT_F16>();
}

int onhip_cache_read(const onhip_cache_desc_t *c, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale,
                     const int32_t *table, long long table_stride, int32_t table_pages, const int32_t *lengths,
                     int32_t batch, int32_t tokens, void *k_out, const long long k_out_strides[3], void *v_out, const long long v_out_strides[3],
                     void *stream) {
    ReadParams p;
    int dt, rc = cache_shape("cache read", c, &p.c, &dt);
    if (!rc) rc = cache_memory("cache read", c, k_cache, v_cache, k_scale, v_scale, &p.c);
    if (rc) return rc;
    if (batch < 1 || tokens < 1 || table_pages < 0 || table_stride < 0) return set_error(ONHIP_ERR_ARG, "cache read: bad shape");
    if (batch > 32767 || c->kv_heads > 65535) return set_error(ONHIP_ERR_ARG, "cache read: %d sequences of %d heads", batch, c->kv_heads);
    if (tokens > (1 << 30)) return set_error(ONHIP_ERR_ARG, "cache read: %d tokens", tokens);
    if ((table_pages > 0 && !table) || !lengths || !k_out || !v_out || !k_out_strides || !v_out_strides) return set_error(ONHIP_ERR_ARG, "cache read: null pointer");
    if (reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16) return set_error(ONHIP_ERR_ARG, "cache read: results must be 16-byte aligned");
    if (k_out == v_out) return set_error(ONHIP_ERR_ARG, "cache read: one result for k and v");
    const long long *strides[2] = {k_out_strides, v_out_strides};
    const int extent[3] = {batch, c->kv_heads, tokens};
    for (int t = 0; t < 2; ++t)
        for (int i = 0; i < 3; ++i) {
            p.os[t][i] = 0;   // a stride that is never stepped over
            if (extent[i] == 1) continue;
            if (strides[t][i] % 8 || strides[t][i] < c->head_dim)
                return set_error(ONHIP_ERR_ARG, "cache read: strides of the results must be multiples of 8, at least the head dimension");
            p.os[t][i] = strides[t][i];
        }
    for (int t = 0; t < 2; ++t)
        if (!rows_apart(extent, strides[t], c->head_dim)) return set_error(ONHIP_ERR_ARG, "cache read: rows of a result overlap");
    if (k_out == k_cache || k_out == v_cache || v_out == k_cache || v_out == v_cache) return set_error(ONHIP_ERR_ARG, "cache read: one memory for a result and the cache");
    p.k_out = reinterpret_cast<unsigned short *>(k_out);
    p.v_out = reinterpret_cast<unsigned short *>(v_out);
    p.table = table;
    p.lengths = lengths;
    p.table_stride = table_stride;
    p.table_pages = table_pages;
    p.batch = batch;
    p.kv_heads = c->kv_heads;
    p.tokens = tokens;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto by_size = [&]<int DT>() {
        if (c->head_dim == 64) return c->quantised ? read_launch<DT, 64, true>(p, st) : read_launch<DT, 64, false>(p, st);
        return c->quantised ? read_launch<DT, 128, true>(p, st) : read_launch<DT, 128, false>(p, st);
    };
    return dt == DT_BF16 ? by_size.template operator()<DT_BF16>() : by_size.template operator()<DT_F16>();
}

}  // extern "C"
