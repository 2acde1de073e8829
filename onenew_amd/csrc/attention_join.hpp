// Attention whose keys were shared out among workgroups: every part leaves its unnormalised result, its largest score m (in units of the
// exponential base 2) and the sum l of its exponentials; the join is sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
#pragma once

#include "igemm_kernel.hpp"

namespace onhip {

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
