// What the attention kernels on long sequences share: the cap of scores, and the join of parts.
//
// Attention whose keys were shared out among workgroups: every part leaves its unnormalised result, its largest score m (in units of the
// exponential base 2) and the sum l of its exponentials; the join is sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  A part without a score above
// minus infinity leaves no result, and l = 0 where the row sees no key, 1 where it does: where no part has one, zeros and NaN.
#pragma once

#include "igemm_kernel.hpp"

namespace onhip {

// s -> cap tanh(s scale / cap) log2(e).  Up to half of the cap, where most scores are, tanh(x) = x P(x^2), P of degree 3 fitted to the smallest largest
// error, 1.6 10^-7 in fp32 (2.4 10^-6 of x where x is small, so that a cap far above the scores leaves them alone): 24 cycles a score.  Above it
// 1 - 2 / (e^2x + 1), off by 2^-23 of the cap: 44 cycles.  Each score by its own size: a row's bits do not depend on the rows beside it.
struct Cap {
    float cap2, to_x, to_exp;        // cap log2(e), 0 for none; scale / cap; twice that times log2(e)
    float tanh0, tanh1, tanh2, tanh3;   // cap2 times the coefficients of P
};
inline Cap make_cap(float scale, float cap) {
    Cap c = {cap * 1.44269504088896340736f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (!(cap > 0.0f)) return c;
    c.to_x = scale / cap;
    c.to_exp = c.to_x * 2.0f * 1.44269504088896340736f;
    c.tanh0 = c.cap2 * 0.999997675f;
    c.tanh1 = c.cap2 * -0.333206564f;
    c.tanh2 = c.cap2 * 0.131451443f;
    c.tanh3 = c.cap2 * -0.0433724485f;
    return c;
}
// scale and cap (0: none) whose quotient and products with log2(e) keep clear of the ends of fp32's range
inline bool cap_fits(float scale, float cap) {
    const float s = fabsf(scale);
    if (!(s < 1e30f) || !(cap >= 0.0f) || !(cap < 1e30f)) return false;
    return cap == 0.0f || s == 0.0f || (s / cap > 1e-30f && s / cap < 1e30f);
}
// a slope of 10^28 leaves one key to a row as a larger one does, and times a distance stays in fp32's range
__device__ __forceinline__ float slope_within(float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -1e28f, 1e28f); }
__device__ __forceinline__ float cap_near(const Cap &c, float s) {
    const float x = s * c.to_x, y = x * x;
    return x * __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c.tanh3, y, c.tanh2), y, c.tanh1), y, c.tanh0);
}
__device__ __forceinline__ float cap_any(const Cap &c, float s) {
    const float e = __builtin_amdgcn_exp2f(s * c.to_exp), far = __builtin_fmaf(-2.0f * c.cap2, __builtin_amdgcn_rcpf(e + 1.0f), c.cap2);
    return fabsf(s * c.to_x) <= 0.5f ? cap_near(c, s) : far;
}
template <int N> __device__ __forceinline__ void cap_scores(const Cap &c, float (&s)[N]) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(s[i] * c.to_x));
    if (!__any(most > 0.5f)) {   // uniform: no exponential at all
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = cap_near(c, s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = cap_any(c, s[i]);
    }
}

// parts of one result row lie one behind the other: o[row][splits][HD], ml[row][splits][2]
struct JoinParams {
    const float *o, *ml;
    unsigned short *out;
    long long os[3];       // elements: (batch, head, token); a row is ((batch * heads) + head) * tokens + token
    int heads, tokens, splits;
    long long rows;
};

// floats of the parts of `rows` rows
inline size_t join_bytes(long long rows, int splits, int hd) { return splits > 1 ? (size_t) rows * splits * (hd + 2) * 4 : 0; }

int attention_join_launch(int dt, int hd, const JoinParams &p, hipStream_t stream);

}  // namespace onhip
