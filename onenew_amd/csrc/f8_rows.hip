// Rows on their way into a product in 8-bit floating point: the root-mean-square norm of a row plus its residual, and rows, gated rows and weights as e4m3
// with scales (f8_common.hpp).
//
//   norm:   h = x + r,  sum = round(h),  y = h / sqrt(mean(h^2) + eps) * w
//   gated:  y = g / (1 + e^-g) * u, g and u the two halves of a row
// in fp32; y goes out in x's type or as e4m3 and scales.  What leaves fp32's range on the way and not in the result has a way of its own: squares of a row, the exponential of a low gate.
//
// A lane has eight consecutive channels (16 bytes of a 16-bit type in, 8 bytes of e4m3 out), sixteen lanes a block of 128: its largest magnitude goes from
// lane to lane in the vector pipe.  Every operand is read once and every result written once (rows of the norm past 16384 channels are read twice).
//
// Bound by memory, or by a launch's few microseconds where rows are few: the norm of 8191 bf16 rows of 4096 with residual and sum 235 MB in 49 us (4.8 TB/s; a large copy reaches 4.9 to 5.4),
// 4001 gated rows of 11008 221 MB in 40 (part of it from the last-level cache), 8192 fp16 rows of 4096 102 MB in 17 (as well), fp32 weights of 11008 x 4096 226 MB in 42.
#include "f8_common.hpp"

namespace onhip {

struct NormParams {
    const char *x, *res;
    const float *weight;
    char *out, *sum;
    float *scale;
    long long xs, rs, os, us;    // bytes between rows: x, residual, result, sum
    long long ss[2];             // floats between rows and blocks of the scales
    int rows, n;
    float eps;
};

// WAVES wavefronts a row (one: four rows a workgroup), NI groups of eight channels a lane, so that a row stays in registers between its sum and its result; a row longer than that (LONG) is read twice.
// One row's time is its chain of loads, sum and store: 4096 channels take four wavefronts 3 us with the launch
template <int DT, bool F8, int WAVES, int NI, bool LONG>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void rms_norm_kernel(const NormParams p) {
    constexpr int SIZE = element_bytes<DT>, STEP = 512 * WAVES;
    __shared__ float part[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long row = WAVES == 1 ? f8_group() * 4 + wave : f8_group();
    if (row >= p.rows) return;   // all of a workgroup, or WAVES == 1, where nothing below synchronises
    const char *x = p.x + row * p.xs, *res = p.res ? p.res + row * p.rs : nullptr;
    const int first = (WAVES == 1 ? 0 : wave) * 512 + lane * 8;

    auto load = [&](int at, float (&h)[8]) __attribute__((always_inline)) {
        load8<DT>(x + (long long) at * SIZE, p.n - at, h);
        if (res) {
            float r[8];
            load8<DT>(res + (long long) at * SIZE, p.n - at, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] += r[j];
        }
    };
    float h[NI][8];
    if constexpr (!LONG) {
#pragma unroll
        for (int i = 0; i < NI; ++i) load(first + i * STEP, h[i]);
    }
    // sum of (h by)^2 over the row
    auto squares = [&](float by) __attribute__((always_inline)) {
        float total = 0.0f;
        auto add = [&](const float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) total = __builtin_fmaf(v[j] * by, v[j] * by, total);
        };
        if constexpr (LONG) {
            for (int at = first; at < p.n; at += STEP) {
                load(at, h[0]);
                add(h[0]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) add(h[i]);
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
        if constexpr (WAVES > 1) {
            __syncthreads();
            if (lane == 0) part[wave] = total;
            __syncthreads();
            total = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) total += part[w];
        }
        return total;
    };
    // a row whose squares leave fp32's range is scaled by a power of two (without eps, or one below 2^-80, one of small numbers as well)
    float total = squares(1.0f), by = 1.0f;
    if (!(total < INFINITY) || (total < 0x1p-100f && p.eps < 0x1p-80f)) {   // uniform over the row
        by = total < 1.0f ? 0x1p100f : 0x1p-80f;
        total = squares(by);
    }
    const float root = rsqrtf(total / (float) p.n + p.eps * by * by);
    // the small one of a value's two factors behind the other: a small value of a row that is scaled down, times 2^-80 at first, would lose bits as a subnormal number
    const float once = by < 1.0f ? root : by, then = by < 1.0f ? by : root;

    auto finish = [&](int at, const float (&v)[8]) __attribute__((always_inline)) {
        const int left = p.n - at;
        if (p.sum && left > 0) store8<DT>(p.sum + row * p.us + (long long) at * SIZE, left, v);
        float y[8], w[8];
        if (p.weight) load8<DT_F32>(reinterpret_cast<const char *>(p.weight + at), left, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = v[j] * once * then * (p.weight ? w[j] : 1.0f);
        if constexpr (F8) {
            const float s = f8_scale(block_top(y));
            if (left > 0) {
                f8_store(p.out + row * p.os + at, left, f8_pack(y, s));
                if (lane % 16 == 0) p.scale[row * p.ss[0] + at / F8_BLOCK * p.ss[1]] = s;
            }
        } else {
            if (left > 0) store8<DT>(p.out + row * p.os + (long long) at * SIZE, left, y);
        }
    };
    if constexpr (LONG) {
        for (int base = first - lane * 8; base < p.n; base += STEP) {   // all lanes of a block, also behind the row's end
            load(base + lane * 8, h[0]);
            finish(base + lane * 8, h[0]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (first - lane * 8 + i * STEP < p.n) finish(first + i * STEP, h[i]);
    }
}

struct RowsParams {
    const char *x;
    char *out;
    float *scale;
    long long xs, os;     // bytes between rows
    long long ss[2];      // floats
    int n, blocks;        // channels of a result row, its blocks of 128
    unsigned items;       // rows x blocks
    Div31 by_blocks;
};

// sixteen lanes a block of 128, four blocks a wavefront
template <int DT, bool GATED>
__global__ __launch_bounds__(256) void f8_rows_kernel(const RowsParams p) {
    constexpr int SIZE = element_bytes<DT>;
    const unsigned item = (unsigned) f8_group() * 16 + threadIdx.x / 16;
    if (item >= p.items) return;   // sixteen lanes at a time, and what follows is between those
    const long long row = div31(item, p.by_blocks);
    const int block = (int) (item - (unsigned) row * p.blocks), at = block * F8_BLOCK + (threadIdx.x & 15) * 8, left = p.n - at;
    float y[8];
    load8<DT>(p.x + row * p.xs + (long long) at * SIZE, left, y);
    if constexpr (GATED) {
        constexpr float LOG2E = 1.44269504088896340736f;
        float u[8], z[8], lowest = 0.0f;
        load8<DT>(p.x + row * p.xs + ((long long) p.n + at) * SIZE, left, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // e^-|g|, so that neither side leaves fp32's range; off by 1.25 |g| 2^-24 of itself, the exponent's rounding and its constant's (an exponent in two parts changed one e4m3 of 25 million)
            const float g = y[j], e = __builtin_amdgcn_exp2f(fabsf(g) * -LOG2E), d = 1.0f + e;
            float inv = __builtin_amdgcn_rcpf(d);
            inv = __builtin_fmaf(__builtin_fmaf(-d, inv, 1.0f), inv, inv);
            z[j] = (g < 0.0f ? g * e : g) * inv * u[j];
            lowest = fminf(lowest, g);
        }
        if (lowest < -87.0f) {
            // The instruction gives zero for a subnormal e, from g = -87.34 on, where g e u need not be small: g e^g u with e^g in three parts, the last two the square root of what is
            // below 2^-120 (1 + e^g is 1 there).  Below -1000 it is zero for every u
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float g = fmaxf(y[j], -1000.0f), a = g * LOG2E, high = fmaxf(a, -120.0f), low = __builtin_amdgcn_exp2f(0.5f * (a - high));
                if (y[j] < -87.0f && y[j] > -INFINITY) z[j] = g * __builtin_amdgcn_exp2f(high) * u[j] * low * low;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = z[j];
    }
    const float s = f8_scale(block_top(y));
    if (left > 0) f8_store(p.out + row * p.os + at, left, f8_pack(y, s));
    if ((threadIdx.x & 15) == 0) p.scale[row * p.ss[0] + block * p.ss[1]] = s;
}

struct WeightsParams {
    const char *x;
    char *out;
    float *scale;
    long long xs, os;
    long long ss[2];
    int rows, n, blocks, scale_rows;
};

// a workgroup a block of 128 x 128: sixteen lanes have 128 channels of eight of its rows
template <int DT>
__global__ __launch_bounds__(256) void f8_weights_kernel(const WeightsParams p) {
    __shared__ float part[4];
    const unsigned group = (unsigned) f8_group();
    const int tile = (int) (group / (unsigned) p.blocks), block = (int) (group % (unsigned) p.blocks);
    if (tile >= p.scale_rows) return;
    const int at = block * F8_BLOCK + (threadIdx.x & 15) * 8, left = p.n - at;
    const long long first = (long long) tile * F8_BLOCK + threadIdx.x / 16;
    float y[8][8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long row = first + 16 * i;
        load8<DT>(p.x + row * p.xs + (long long) at * element_bytes<DT>, row < p.rows ? left : 0, y[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, block_top(y[i]));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = top;
    __syncthreads();
    const float s = f8_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long row = first + 16 * i;
        if (row < p.rows && left > 0) f8_store(p.out + row * p.os + at, left, f8_pack(y[i], s));
    }
    if (threadIdx.x == 0) p.scale[tile * p.ss[0] + block * p.ss[1]] = s;
}

// ---- checks and launches -------------------------------------------------------------------------------------------

// a matrix of `rows` rows of `n` elements of `size` bytes: its row stride in bytes, 0 where there is one row
static int row_step(const char *what, const char *name, const void *at, int rows, long long n, long long stride, int size, bool written, long long *step) {
    *step = 0;
    if (!at) return set_error(ONHIP_ERR_ARG, "%s: null %s", what, name);
    if (misaligned(at, (uintptr_t) size)) return set_error(ONHIP_ERR_ARG, "%s: misaligned %s", what, name);
    if (rows <= 1) return ONHIP_OK;
    if (stride < (written ? n : 0) || stride > (1LL << 40)) return set_error(ONHIP_ERR_ARG, "%s: a row stride of %lld for %s", what, stride, name);
    *step = stride * size;
    return ONHIP_OK;
}

// e4m3 rows and scales as results
static int f8_result(const char *what, void *q, long long q_stride, float *scale, const long long *scale_strides, int rows, int scale_rows, int n, long long *os, long long *ss) {
    const int blocks = (n + F8_BLOCK - 1) / F8_BLOCK;
    if (int rc = row_step(what, "result", q, rows, n, q_stride, 1, true, os)) return rc;
    if (misaligned(q, 16) || *os % 16) return set_error(ONHIP_ERR_ARG, "%s: e4m3 rows must be 16-byte aligned", what);
    if (!scale || !scale_strides || misaligned(scale, 4)) return set_error(ONHIP_ERR_ARG, "%s: null or misaligned scales", what);
    const int extent[2] = {scale_rows, blocks};
    for (int i = 0; i < 2; ++i) {
        ss[i] = extent[i] == 1 ? 0 : scale_strides[i];
        if (extent[i] > 1 && (ss[i] < 1 || ss[i] > (1LL << 40))) return set_error(ONHIP_ERR_ARG, "%s: bad scale strides", what);
    }
    if (!rows_apart(extent, scale_strides, 1)) return set_error(ONHIP_ERR_ARG, "%s: scales overlap", what);
    return ONHIP_OK;
}

template <int DT, bool F8>
static int norm_launch(const NormParams &p, hipStream_t stream) {
    const unsigned rows = (unsigned) p.rows;
    auto go = [&]<int WAVES, int NI, bool LONG>() {
        hipLaunchKernelGGL((rms_norm_kernel<DT, F8, WAVES, NI, LONG>), f8_grid(WAVES == 1 ? (rows + 3) / 4 : rows), dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, stream, p);
    };
    if (p.n <= 512) go.template operator()<1, 1, false>();
    else if (p.n <= 2048) go.template operator()<4, 1, false>();
    else if (p.n <= 4096) go.template operator()<4, 2, false>();
    else if (p.n <= 8192) go.template operator()<8, 2, false>();
    else if (p.n <= 16384) go.template operator()<16, 2, false>();
    else go.template operator()<16, 1, true>();
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

}  // namespace onhip

using namespace onhip;

extern "C" {

int onhip_rms_norm(const onhip_norm_desc_t *d, const void *x, const void *residual, const float *weight, void *out, float *out_scale, void *sum, void *stream) {
    const char *what = "rms norm";
    NormParams p = {};
    int dt;
    if (!d || d->rows < 1 || d->channels < 1) return set_error(ONHIP_ERR_ARG, "%s: bad shape", what);
    if (d->channels > (1 << 30)) return set_error(ONHIP_ERR_ARG, "%s: %d channels", what, d->channels);
    if (!element_type(d->compute, &dt)) return set_error(ONHIP_ERR_ARG, "%s: unknown type %d", what, d->compute);
    if (d->f8 != 0 && d->f8 != 1) return set_error(ONHIP_ERR_ARG, "%s: f8 = %d", what, d->f8);
    if (!(d->eps >= 0.0f)) return set_error(ONHIP_ERR_ARG, "%s: eps must not be negative", what);
    if (sum && !residual) return set_error(ONHIP_ERR_ARG, "%s: a sum without a residual", what);
    const int size = bytes_of(dt);
    int rc = row_step(what, "x", x, d->rows, d->channels, d->x_stride, size, false, &p.xs);
    if (!rc && residual) rc = row_step(what, "residual", residual, d->rows, d->channels, d->residual_stride, size, false, &p.rs);
    if (!rc && sum) rc = row_step(what, "sum", sum, d->rows, d->channels, d->sum_stride, size, true, &p.us);
    if (rc) return rc;
    if (weight && misaligned(weight, 4)) return set_error(ONHIP_ERR_ARG, "%s: misaligned weight", what);
    if (d->f8) rc = f8_result(what, out, d->out_stride, out_scale, d->scale_strides, d->rows, d->rows, d->channels, &p.os, p.ss);
    else rc = row_step(what, "result", out, d->rows, d->channels, d->out_stride, size, true, &p.os);
    if (rc) return rc;
    const long long row = (long long) d->channels * size, blocks = (d->channels + F8_BLOCK - 1) / F8_BLOCK;
    const Span of_x = {static_cast<const char *>(x), p.xs, row, d->rows}, of_r = {static_cast<const char *>(residual), p.rs, row, d->rows},
               of_sum = {static_cast<const char *>(sum), p.us, row, d->rows}, of_w = {reinterpret_cast<const char *>(weight), 0, 4LL * d->channels, 1},
               of_out = {static_cast<const char *>(out), p.os, d->f8 ? (long long) d->channels : row, d->rows},
               of_scale = scale_span(d->f8 ? out_scale : nullptr, p.ss, d->rows, (int) blocks);
    if (!apart(of_out, of_sum) || !apart(of_out, of_scale) || !apart(of_sum, of_scale)) return set_error(ONHIP_ERR_ARG, "%s: one memory for two results", what);
    // a lane writes an element when it has read x and the residual there: results of their type may take their places, but not the weight's, which is read behind the sum's store and by every row
    auto fits = [&](const Span &result, bool like) {
        for (const Span &from : {of_x, of_r})
            if (!apart(result, from) && !(like && same(result, from))) return false;
        return apart(result, of_w);
    };
    if (!fits(of_out, !d->f8) || !fits(of_sum, true) || !fits(of_scale, false)) return set_error(ONHIP_ERR_ARG, "%s: a result lies over an operand", what);
    p.x = static_cast<const char *>(x);
    p.res = static_cast<const char *>(residual);
    p.weight = weight;
    p.out = static_cast<char *>(out);
    p.sum = static_cast<char *>(sum);
    p.scale = out_scale;
    p.rows = d->rows;
    p.n = d->channels;
    p.eps = d->eps;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto by_kind = [&]<int DT>() { return d->f8 ? norm_launch<DT, true>(p, st) : norm_launch<DT, false>(p, st); };
    return dt == DT_F32 ? by_kind.template operator()<DT_F32>() : dt == DT_BF16 ? by_kind.template operator()<DT_BF16>() : by_kind.template operator()<DT_F16>();
}

int onhip_f8_from_rows(const onhip_f8_rows_desc_t *d, const void *x, void *q, float *scale, void *stream) {
    const char *what = "rows to e4m3";
    int dt;
    if (!d || d->rows < 1 || d->channels < 1) return set_error(ONHIP_ERR_ARG, "%s: bad shape", what);
    if (d->channels > (1 << 30)) return set_error(ONHIP_ERR_ARG, "%s: %d channels", what, d->channels);
    if (!element_type(d->compute, &dt)) return set_error(ONHIP_ERR_ARG, "%s: unknown type %d", what, d->compute);
    if (d->form != ONHIP_F8_ROWS && d->form != ONHIP_F8_GATED && d->form != ONHIP_F8_WEIGHTS) return set_error(ONHIP_ERR_ARG, "%s: form %d", what, d->form);
    const bool weights = d->form == ONHIP_F8_WEIGHTS, gated = d->form == ONHIP_F8_GATED;
    const int blocks = (d->channels + F8_BLOCK - 1) / F8_BLOCK, size = bytes_of(dt);
    const int scale_rows = weights ? (int) (((long long) d->rows + F8_BLOCK - 1) / F8_BLOCK) : d->rows;
    long long xs, os, ss[2];
    int rc = row_step(what, "x", x, d->rows, d->channels * (gated ? 2LL : 1LL), d->x_stride, size, false, &xs);
    if (!rc) rc = f8_result(what, q, d->q_stride, scale, d->scale_strides, d->rows, scale_rows, d->channels, &os, ss);
    if (rc) return rc;
    const Span of_x = {static_cast<const char *>(x), xs, (long long) d->channels * (gated ? 2 : 1) * size, d->rows}, of_q = {static_cast<const char *>(q), os, d->channels, d->rows},
               of_scale = scale_span(scale, ss, scale_rows, blocks);
    if (!apart(of_q, of_x) || !apart(of_scale, of_x) || !apart(of_q, of_scale)) return set_error(ONHIP_ERR_ARG, "%s: results lie over the operand or over each other", what);
    const long long items = (long long) scale_rows * blocks, groups = weights ? items : (items + 15) / 16;
    if (items >= (1LL << 31) - 16) return set_error(ONHIP_ERR_ARG, "%s: too many rows", what);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid = f8_grid(groups);
    const char *from = static_cast<const char *>(x);
    char *to = static_cast<char *>(q);
    if (weights) {
        const WeightsParams p = {from, to, scale, xs, os, {ss[0], ss[1]}, d->rows, d->channels, blocks, scale_rows};
        auto go = [&]<int DT>() {
            hipLaunchKernelGGL((f8_weights_kernel<DT>), grid, dim3(256), 0, st, p);
        };
        dt == DT_F32 ? go.template operator()<DT_F32>() : dt == DT_BF16 ? go.template operator()<DT_BF16>() : go.template operator()<DT_F16>();
    } else {
        const RowsParams p = {from, to, scale, xs, os, {ss[0], ss[1]}, d->channels, blocks, (unsigned) items, make_div31((unsigned) blocks)};
        auto go = [&]<int DT, bool GATED>() {
            hipLaunchKernelGGL((f8_rows_kernel<DT, GATED>), grid, dim3(256), 0, st, p);
        };
        auto by_form = [&]<int DT>() { gated ? go.template operator()<DT, true>() : go.template operator()<DT, false>(); };
        dt == DT_F32 ? by_form.template operator()<DT_F32>() : dt == DT_BF16 ? by_form.template operator()<DT_BF16>() : by_form.template operator()<DT_F16>();
    }
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

}  // extern "C"
