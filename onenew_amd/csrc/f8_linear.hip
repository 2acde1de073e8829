// Product of rows and weights in 8-bit floating point:
//   out[m][n] = sum over blocks b of 128 channels  sa[m][b] sw[n / 128][b] (sum_k a[m][k] w[n][k])  + bias[n]
//
// The inner sums are matrix instructions in bf16, which holds every e4m3, that start at zero; sums over blocks are fp32, a fused multiply-add a
// value.  (The instructions on e4m3 itself sum eight products at a time with 13 bits below the largest of them.)  Weights are the instruction's rows, so that a
// lane's values belong to one row m: a block has one factor a lane, sa[m] times the wavefront's sw.
//
// Tiles of both operands go from memory straight into LDS, a block of 128 channels of every row a stage, two stages; a row's 16-byte units are exchanged
// as (unit ^ row / 2 % 8), which puts the sixteen rows that are read together on different banks.
#include "f8_common.hpp"

namespace onhip {


struct F8LinearParams {
    const char *a, *w;
    const float *a_scale, *w_scale, *bias;
    char *out;
    long long as, ws, os;            // bytes between rows
    long long a_ss[2], w_ss[2];      // floats between rows and blocks
    int m, n, k;
    int tiles_m, tiles_n;
    bool vec;                        // four results are one aligned store
};

// a unit of 16 bytes of this lane from `voff` behind the descriptor's base (zeros outside) to LDS at `lds` + 16 lane.  In assembly, for the compiler waits for every
// such load in front of any LDS read; the waits are placed by hand.  Nothing else here goes by m0
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, unsigned voff, unsigned soff, unsigned lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" :: "s"(lds), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
#endif
}
__device__ __forceinline__ i32x4 descriptor(const char *base, unsigned bytes) {
    const unsigned long long at = reinterpret_cast<unsigned long long>(base);
    return i32x4{__builtin_amdgcn_readfirstlane((int) (unsigned) at), __builtin_amdgcn_readfirstlane((int) (at >> 32) & 0xffff), __builtin_amdgcn_readfirstlane((int) bytes), (int) RSRC_FLAGS};
}

// eight e4m3 as bf16, which has them all
__device__ __forceinline__ bf16x8 f8_widened(int x, int y) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#else
    return {};
#endif
}

// BN weight rows x BM rows a workgroup, WN x WM wavefronts
template <int DT, int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM) void f8_linear_kernel(const F8LinearParams p) {
    constexpr int WAVES = WN * WM, TN = BN / WN / 32, TM = BM / WM / 32, STAGE = (BN + BM) * 128;
    constexpr int LOADS_N = BN / 8 / WAVES, LOADS_M = BM / 8 / WAVES;   // eight rows a load
    static_assert(BN / WN <= 128 && LOADS_N >= 1 && LOADS_M >= 1, "a wavefront's weights share a scale, and every wavefront loads");
    __shared__ __attribute__((aligned(1024))) char lds[2][STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 31, lh = lane >> 5, wn = wave / WM, wm = wave % WM;
    // tiles: an XCD has a run of them, eight rows of tiles by columns
    int tn, tm;
    {
        const int bid = blockIdx.x, nb = (int) gridDim.x, q = nb >> 3, rem = nb & 7, xcd = bid & 7;
        const int lid = xcd * q + (xcd < rem ? xcd : rem) + (bid >> 3);
        const int group = lid / (8 * p.tiles_n), left = lid - group * 8 * p.tiles_n, high = min(8, p.tiles_m - group * 8);
        tn = left / high;
        tm = group * 8 + left - tn * high;
    }
    const int n0 = tn * BN, m0 = tm * BM;
    const int k_blocks = (p.k + 127) / 128;

    const int rows_n = min(BN, p.n - n0), rows_m = min(BM, p.m - m0), k16 = (p.k + 15) & ~15;
    const char *w_base = p.w + n0 * p.ws, *a_base = p.a + m0 * p.as;
    const unsigned w_bytes = (unsigned) ((rows_n - 1) * p.ws + k16), a_bytes = (unsigned) ((rows_m - 1) * p.as + k16);
    unsigned w_off[LOADS_N], a_off[LOADS_M];
    const int lrow = lane / 8;
#pragma unroll
    for (int t = 0; t < LOADS_N; ++t) {
        const int row = (wave * LOADS_N + t) * 8 + lrow;
        w_off[t] = row < rows_n ? (unsigned) (row * p.ws) + ((lane % 8) ^ (row / 2 % 8)) * 16 : OOB;
    }
#pragma unroll
    for (int t = 0; t < LOADS_M; ++t) {
        const int row = (wave * LOADS_M + t) * 8 + lrow;
        a_off[t] = row < rows_m ? (unsigned) (row * p.as) + ((lane % 8) ^ (row / 2 % 8)) * 16 : OOB;
    }
    const i32x4 rw = descriptor(w_base, w_bytes), ra = descriptor(a_base, a_bytes);
    const unsigned lds0 = (unsigned) (size_t) (__attribute__((address_space(3))) char *) &lds[0][0];
    auto issue = [&](int kb, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < LOADS_N; ++t) load_to_lds(rw, w_off[t], (unsigned) kb * 128u, lds0 + buf * STAGE + (wave * LOADS_N + t) * 1024);
#pragma unroll
        for (int t = 0; t < LOADS_M; ++t) load_to_lds(ra, a_off[t], (unsigned) kb * 128u, lds0 + buf * STAGE + BN * 128 + (wave * LOADS_M + t) * 1024);
    };

    // factors of a block: this lane's rows m, and the wavefront's weights
    const int m_wave = m0 + wm * (BM / WM), n_wave = n0 + wn * (BN / WN);
    const float *sw = p.w_scale + (n_wave < p.n ? n_wave / 128 : 0) * p.w_ss[0];
    const float *sa[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) sa[t] = p.a_scale + (long long) min(m_wave + t * 32 + li, p.m - 1) * p.a_ss[0];

    f32x16 acc[TN][TM] = {};
    issue(0, 0);
    for (int kb = 0; kb < k_blocks; ++kb) {
        const int buf = kb & 1;
        float s[TM];
#pragma unroll
        for (int t = 0; t < TM; ++t) s[t] = sa[t][kb * p.a_ss[1]] * sw[kb * p.w_ss[1]];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this stage is there, and everybody has read the other one
        __syncthreads();
        char *stage = lds[buf];
        const int there = p.k - kb * 128;
        if (there < 128) {   // the last block: nothing behind a row's end takes part
            for (int i = threadIdx.x; i < (BN + BM) * 8; i += 64 * WAVES) {
                const int row = i / 8, unit = (i % 8) ^ (row / 2 % 8), keep = there - unit * 16;
                if (keep >= 16) continue;
                unsigned *at = reinterpret_cast<unsigned *>(stage + i * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int bytes = keep - 4 * j;
                    at[j] = bytes >= 4 ? at[j] : bytes <= 0 ? 0u : at[j] & (0xffffffffu >> (32 - 8 * bytes));
                }
            }
            __syncthreads();
        }
        if (kb + 1 < k_blocks) issue(kb + 1, buf ^ 1);
        // this lane's 16 bytes of a row: units 2 i and 2 i + 1 are the two halves of the wavefront's
        auto operand = [&](int row, int i, bf16x8 (&x)[2]) __attribute__((always_inline)) {
            const i32x4 q = *reinterpret_cast<const i32x4 *>(stage + row * 128 + ((2 * i + lh) ^ (row / 2 % 8)) * 16);
            x[0] = f8_widened(q[0], q[1]);
            x[1] = f8_widened(q[2], q[3]);
        };
        f32x16 part[TN][TM] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 a[TN][2], b[TM][2];
#pragma unroll
            for (int t = 0; t < TM; ++t) operand(BN + wm * (BM / WM) + t * 32 + li, i, b[t]);
#pragma unroll
            for (int u = 0; u < TN; ++u) operand(wn * (BN / WN) + u * 32 + li, i, a[u]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int u = 0; u < TN; ++u)
#pragma unroll
                    for (int t = 0; t < TM; ++t) part[u][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[u][h], b[t][h], part[u][t], 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < TN; ++u)
#pragma unroll
            for (int t = 0; t < TM; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[u][t][r] = __builtin_fmaf(part[u][t][r], s[t], acc[u][t][r]);
    }

    // a lane has 4 consecutive n in each of four groups of eight, of row m
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = n_wave + u * 32 + g * 8 + lh * 4;
            float bias[4] = {};
            if (p.bias)
#pragma unroll
                for (int j = 0; j < 4; ++j) bias[j] = n + j < p.n ? p.bias[n + j] : 0.0f;
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                const int m = m_wave + t * 32 + li;
                if (m >= p.m || n >= p.n) continue;
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = acc[u][t][g * 4 + j] + bias[j];
                char *at = p.out + m * p.os + (long long) n * element_bytes<DT>;
                if (p.vec && n + 4 <= p.n) {
                    if constexpr (DT == DT_F32) *reinterpret_cast<float4 *>(at) = make_float4(v[0], v[1], v[2], v[3]);
                    else *reinterpret_cast<uint2 *>(at) = make_uint2(pack_h16<DT>(v[0], v[1]), pack_h16<DT>(v[2], v[3]));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n + j < p.n) {
                            if constexpr (DT == DT_F32) reinterpret_cast<float *>(at)[j] = v[j];
                            else reinterpret_cast<unsigned short *>(at)[j] = (unsigned short) pack_h16<DT>(v[j], 0.0f);
                        }
                }
            }
        }
}

template <int DT, int BN, int BM, int WN, int WM> static int linear_launch(F8LinearParams p, hipStream_t stream) {
    p.tiles_n = (p.n + BN - 1) / BN;
    p.tiles_m = (p.m + BM - 1) / BM;
    hipLaunchKernelGGL((f8_linear_kernel<DT, BN, BM, WN, WM>), dim3((unsigned) p.tiles_n * p.tiles_m), dim3(64 * WN * WM), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

static bool off(const void *at, uintptr_t to) { return reinterpret_cast<uintptr_t>(at) % to != 0; }

static int linear_check(const onhip_f8_linear_desc_t *d, int *dt) {
    const char *what = "e4m3 product";
    if (!d || d->rows < 1 || d->outputs < 1 || d->channels < 1) return set_error(ONHIP_ERR_ARG, "%s: bad shape", what);
    if (!element_type(d->compute, dt)) return set_error(ONHIP_ERR_ARG, "%s: unknown type %d", what, d->compute);
    if (d->channels > (1 << 22)) return set_error(ONHIP_ERR_ARG, "%s: %d channels (up to 2^22)", what, d->channels);
    // byte offsets within a tile stay below 2^31
    const long long most = 1LL << 22;
    if (d->rows > 1 && (d->a_stride < d->channels || d->a_stride > most || d->a_stride % 16)) return set_error(ONHIP_ERR_ARG, "%s: rows %lld bytes apart (a multiple of 16, up to 2^22)", what, d->a_stride);
    if (d->outputs > 1 && (d->w_stride < d->channels || d->w_stride > most || d->w_stride % 16)) return set_error(ONHIP_ERR_ARG, "%s: weights %lld bytes apart (a multiple of 16, up to 2^22)", what, d->w_stride);
    if (d->rows > 1 && (d->out_stride < d->outputs || d->out_stride > (1LL << 40))) return set_error(ONHIP_ERR_ARG, "%s: results %lld elements apart", what, d->out_stride);
    for (int i = 0; i < 2; ++i)
        if (d->a_scale_strides[i] < 0 || d->a_scale_strides[i] > (1LL << 31) || d->w_scale_strides[i] < 0 || d->w_scale_strides[i] > (1LL << 31))
            return set_error(ONHIP_ERR_ARG, "%s: bad scale strides", what);
    return ONHIP_OK;
}

}  // namespace onhip

using namespace onhip;

extern "C" {

int onhip_linear_f8(const onhip_f8_linear_desc_t *d, const void *a, const float *a_scale, const void *w, const float *w_scale, const float *bias, void *out, void *stream) {
    const char *what = "e4m3 product";
    int dt;
    if (int rc = linear_check(d, &dt)) return rc;
    if (!a || !a_scale || !w || !w_scale || !out) return set_error(ONHIP_ERR_ARG, "%s: null pointer", what);
    if (off(a, 16) || off(w, 16)) return set_error(ONHIP_ERR_ARG, "%s: rows and weights must be 16-byte aligned", what);
    const int size = bytes_of(dt);
    if (off(a_scale, 4) || off(w_scale, 4) || off(bias, 4) || off(out, (uintptr_t) size)) return set_error(ONHIP_ERR_ARG, "%s: misaligned scales, bias or result", what);
    F8LinearParams p = {};
    p.a = static_cast<const char *>(a);
    p.w = static_cast<const char *>(w);
    p.a_scale = a_scale;
    p.w_scale = w_scale;
    p.bias = bias;
    p.out = static_cast<char *>(out);
    p.m = d->rows;
    p.n = d->outputs;
    p.k = d->channels;
    p.as = d->rows > 1 ? d->a_stride : 0;
    p.ws = d->outputs > 1 ? d->w_stride : 0;
    p.os = d->rows > 1 ? d->out_stride * size : 0;
    for (int i = 0; i < 2; ++i) {
        p.a_ss[i] = d->a_scale_strides[i];
        p.w_ss[i] = d->w_scale_strides[i];
    }
    p.vec = !off(out, 4 * (uintptr_t) size) && p.os % (4 * size) == 0;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto go = [&]<int DT>() { return linear_launch<DT, 128, 128, 2, 2>(p, st); };
    return dt == DT_F32 ? go.template operator()<DT_F32>() : dt == DT_BF16 ? go.template operator()<DT_BF16>() : go.template operator()<DT_F16>();
}

}  // extern "C"
