// Attention of prompts:  s_ij = cap tanh(scale q_i.k_j / cap) - slope |P_i - j|,  out_i = Softmax(s_i) v  over the keys that row i sees, in one
// pass over the keys with the running maximum and sum of a softmax; P_i = i + q_offset is the query's place among the keys.
//
// What a row sees is an interval of keys, whatever the mask: causal (j <= P), a window (P - j < window) and the row's own pair
// [begin, end) (documents of a packed batch, prefixes, lengths) are intersected once.  Tiles outside the union of a workgroup's intervals
// are not touched, tiles inside the intersection of a wavefront's are computed without a mask.
//
// Rows: a workgroup has 64, 128 or 256 rows of one key-value head, (token, head of the group) with the head running fastest, so that heads that share
// keys share the tiles that are staged.  A wavefront has 32 of them and computes the transposed scores S^T = k q^T with
// v_mfma_f32_32x32x16, so a lane owns one row and, per 32 keys, the 16 keys 8 (r / 4) + 4 (lane / 32) + r % 4; its softmax is the lane's own, and the
// probabilities feed out^T = v^T P^T from the registers they are in.  Tiles of 64 keys of k and v go through LDS in two buffers, v
// transposed on its way out by the transposing read.
//
// Rounded to the 16-bit type before the second product: 2^(s - m) times a constant, at most 2^8 of it (the reference point m follows a row's maximum when that is
// 2^8 above it, so that most tiles leave the sums alone).  Scores, maxima, sums and products' sums are fp32.
//
// What bounds it: per tile of 64 keys the matrix instructions take 1024 cycles of a SIMD, the softmax's vector instructions as many (half of the exponentials run
// between the second product's matrix instructions), LDS 1300 for operands and staging; two wavefronts a SIMD overlap them to half of the
// time, at a clock that falls under them (1.74 GHz): 8192 causal tokens of 32 heads of 128 on 8 in bf16 500 to 535 us, 1.02 to 1.10 PFLOP/s where a large library
// product reaches 1.2 (540 to 565 with a tile staged for 128 rows, not 256).  Capped scores add a third to the vector work: 2 x 4001 tokens of 16 heads on 8 in a window of 1024, fp16, 98 to 102 us.  Short rows are bound by a
// workgroup's chain of tiles: 2 x 4096 tokens of 16 heads of 64 in documents of about 450, with a bias, 38 to 47 us (their 67 MB take 13).  Tiles of 32 keys with
// three workgroups a compute unit, eight operands ahead, a higher wave priority in the products, and 256 rows on four buffers with a barrier every second tile were level.
#include "attention_join.hpp"
#include "kv_common.hpp"

namespace onhip {

struct MaskedParams {
    const unsigned short *q, *k, *v;
    unsigned short *out;
    long long qs[3], ks[3], vs[3], os[3];   // elements: (batch, head, token)
    const int *ranges;
    const float *slopes;
    int batch, q_heads, kv_heads, group, q_tokens, k_tokens, q_offset, causal, window;
    int blocks, splits;                     // row blocks of a key-value head; parts of the keys
    Div31 by_splits, by_heads, by_kv_heads, by_group;
    int spread;                             // the (batch, key-value head) pairs divide evenly among the XCDs
    float scale2, per_scale, far;           // |scale| * log2(e); 1 / |scale|; how far a score may lie above the reference point, 8 in units of the scores
    Cap cap;
    unsigned flip;                          // sign of the scale on q
    float *part_o, *part_ml;
};

// halves of a packed pair that are +inf (0), -inf (1) or NaN (2), as 1.0 of the type; and the pair with all of those zeroed
template <int DT> __device__ __forceinline__ unsigned special_of(unsigned w, int what) {
    constexpr unsigned INF = DT == DT_BF16 ? 0x7f80u : 0x7c00u, ONE = DT == DT_BF16 ? 0x3f80u : 0x3c00u;
    unsigned y = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned x = w >> (16 * h) & 0xffffu;
        const bool is = what == 0 ? x == INF : what == 1 ? x == (INF | 0x8000u) : (x & 0x7fffu) > INF;
        y |= (is ? ONE : 0u) << (16 * h);
    }
    return y;
}
template <int DT> __device__ __forceinline__ unsigned finite_of(unsigned w) {
    constexpr unsigned INF = DT == DT_BF16 ? 0x7f80u : 0x7c00u;
    return ((w & INF) == INF ? 0u : w & 0xffffu) | ((w >> 16 & INF) == INF ? 0u : w & 0xffff0000u);
}

// HOW the scores become exponents.  PLAIN: one fused product takes them there.  BIASED: as that, where every key that counts lies behind its query, so that the
// bias is slope / scale times (the key's number - the row's place): one more matrix instruction, of the number in the tile of 64 (a whole number) and of one
// with the quotient and the rest in three bf16 parts each, all of their 24 bits (documents of 16 heads 40 us, as GENERAL 43).  GENERAL: capped, a
// bias on keys on both sides, or a scale of (nearly) zero; with 64 channels and 128 rows three of its registers are spilled.
enum { PLAIN, BIASED, GENERAL };
// RG: groups of 32 rows of a workgroup.  4 and 8: a wavefront has all keys of a tile for its rows.  2: two wavefronts share the rows, one has the first 32 keys of
// every tile, one the others, and their results are joined in the end.
template <int DT, int HD, int HOW, int RG>
__global__ __launch_bounds__(RG == 8 ? 512 : 256, HD == 64 ? 3 : 2) void attention_masked_kernel(const MaskedParams p) {
    constexpr int KT = 64, NT = RG >= 4 ? 2 : 1, NWV = RG == 8 ? 8 : 4, STEPS = HD / 16, DTILES = HD / 32;
    // probabilities are 2^(s - m + SHIFT): fp16's stay clear of its smallest numbers, a sum of bf16's largest values of fp32's largest
    constexpr float SHIFT = DT == DT_BF16 ? -24.0f : 7.0f;
    constexpr int UNITS = HD / 8, ROWS = 64 / UNITS;           // 16-byte units of a row; rows that a wavefront's load covers
    constexpr int LOADS = KT / ROWS / NWV;                       // loads of a wavefront for its share of a tile of k (or v)
    // Two tiles of k, two of v.  Rows have a pitch by which 16 lanes that take one 16-byte unit of 16 rows of k, and the transposing read's 64 bytes of four rows
    // of v, meet every bank once, and a read's place in its row is a constant of the instruction (units exchanged by row number cost an address register each).
    constexpr int KP = HD * 2 + 16, VP = HD * 2 + 64;
    __shared__ __attribute__((aligned(16))) unsigned char s_kv[2 * KT * (KP + VP)];
    unsigned char *const Vs = s_kv + 2 * KT * KP;
    __shared__ int4 s_span[NWV];
    __shared__ int s_odd;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5, rg = RG >= 4 ? wave : wave >> 1, kh = RG >= 4 ? 0 : wave & 1;
    // item -> (batch, key-value head, row block, part).  Workgroups go to the XCDs in turn; where the heads divide among them, an XCD has whole
    // heads, so that its L2 holds their keys.  The last row blocks, which see most keys under a causal mask, start first; where all items find room at
    // once, a compute unit's second one is from the other end, so that its two (or three) together are no longer than another's.
    int bh, block, split;
    {
        const unsigned pairs = (unsigned) (p.batch * p.kv_heads);
        unsigned local = blockIdx.x, heads = pairs, first = 0, units = 256u;
        if (p.spread) {
            heads = pairs / 8u;
            first = (blockIdx.x & 7u) * heads;
            local = blockIdx.x >> 3;
            units = 32u;
        }
        const unsigned items = heads * (unsigned) (p.blocks * p.splits);
        if (items <= units * (RG == 8 ? 1u : HD == 64 ? 3u : 2u) && local >= units) local = local < 2u * units ? items - 1u - (local - units) : local - units;
        const unsigned per_split = div31(local, p.by_splits);
        split = (int) (local - per_split * (unsigned) p.splits);
        const unsigned from_end = div31(per_split, p.by_heads);
        bh = (int) (first + per_split - from_end * heads);
        block = p.blocks - 1 - (int) from_end;
    }
    const int b = (int) div31((unsigned) bh, p.by_kv_heads), kvh = bh - b * p.kv_heads;

    // rows past the last one are the last one again, and not stored
    const unsigned last_row = (unsigned) p.q_tokens * (unsigned) p.group - 1u, row0 = (unsigned) (block * (32 * RG) + rg * 32);
    const unsigned own_row = min(row0 + (unsigned) li, last_row);
    int token = (int) div31(own_row, p.by_group), head = kvh * p.group + (int) (own_row - (unsigned) token * (unsigned) p.group);
    const int place = token + p.q_offset;
    // q: asked for first, whole rows at a time (a row a lane, each load keeps a compute unit's address path busy for 64 cycles)
    u32x4 qr[32 / ROWS];
#pragma unroll
    for (int i = 0; i < 32 / ROWS; ++i) {
        const unsigned row = min(row0 + (unsigned) (i * ROWS + lane / UNITS), last_row), tk = div31(row, p.by_group);
        qr[i] = *reinterpret_cast<const u32x4 *>(p.q + b * p.qs[0] + (long long) (kvh * p.group + (int) (row - tk * (unsigned) p.group)) * p.qs[1] + tk * p.qs[2] + lane % UNITS * 8);
    }
    auto first_key = [&](int t) __attribute__((always_inline)) { return p.window > 0 ? max(0, t + p.q_offset - p.window + 1) : 0; };
    auto end_key = [&](int t) __attribute__((always_inline)) { return p.causal ? min(p.k_tokens, t + p.q_offset + 1) : p.k_tokens; };
    int lo = first_key(token), hi = end_key(token);
    // the union and the intersection of the rows' intervals, of the wavefront and of the workgroup (no smaller than the union, no larger than the intersection)
    int any_lo, any_hi, all_lo, all_hi, wg_lo, wg_hi, wg_all_lo, wg_all_hi;
    if (p.ranges) {   // uniform
        const int2 rg2 = reinterpret_cast<const int2 *>(p.ranges)[(long long) b * p.q_tokens + token];
        lo = max(lo, rg2.x);
        hi = min(hi, rg2.y);
        if (lo >= hi) lo = hi = 0;   // sees nothing
        any_lo = lo < hi ? lo : 0x7fffffff;
        any_hi = hi;
        all_lo = lo;
        all_hi = hi;
#pragma unroll
        for (int x = 1; x < 32; x *= 2) {
            any_lo = min(any_lo, __shfl_xor(any_lo, x, 64));
            any_hi = max(any_hi, __shfl_xor(any_hi, x, 64));
            all_lo = max(all_lo, __shfl_xor(all_lo, x, 64));
            all_hi = min(all_hi, __shfl_xor(all_hi, x, 64));
        }
        any_lo = __builtin_amdgcn_readfirstlane(any_lo);
        any_hi = __builtin_amdgcn_readfirstlane(any_hi);
        all_lo = __builtin_amdgcn_readfirstlane(all_lo);
        all_hi = __builtin_amdgcn_readfirstlane(all_hi);
        if (lane == 0) s_span[wave] = make_int4(any_lo, any_hi, all_lo, all_hi);
        __syncthreads();
        int4 x = s_span[0], y = s_span[1], z = s_span[2], w = s_span[3];
        if constexpr (RG == 8) {
            auto both = [](const int4 &a, const int4 &b) __attribute__((always_inline)) { return make_int4(min(a.x, b.x), max(a.y, b.y), max(a.z, b.z), min(a.w, b.w)); };
            x = both(x, s_span[4]);
            y = both(y, s_span[5]);
            z = both(z, s_span[6]);
            w = both(w, s_span[7]);
        }
        wg_lo = __builtin_amdgcn_readfirstlane(min(min(x.x, y.x), min(z.x, w.x)));
        wg_hi = __builtin_amdgcn_readfirstlane(max(max(x.y, y.y), max(z.y, w.y)));
        wg_all_lo = __builtin_amdgcn_readfirstlane(max(max(x.z, y.z), max(z.z, w.z)));
        wg_all_hi = __builtin_amdgcn_readfirstlane(min(min(x.w, y.w), min(z.w, w.w)));
    } else {   // both ends grow with the token: the first row's and the last row's are all there is to know
        if (lo >= hi) lo = hi = 0;
        const int t0 = (int) div31(min(row0, last_row), p.by_group), t1 = (int) div31(min(row0 + 31u, last_row), p.by_group);
        any_lo = first_key(t0);
        any_hi = end_key(t1);
        all_lo = first_key(t1);
        all_hi = end_key(t0);
        const unsigned wg_row = (unsigned) (block * (32 * RG));
        const int w0 = (int) div31(wg_row, p.by_group), w1 = (int) div31(min(wg_row + 32u * RG - 1u, last_row), p.by_group);
        wg_lo = first_key(w0);
        wg_hi = end_key(w1);
        wg_all_lo = first_key(w1);
        wg_all_hi = end_key(w0);
    }
    if (tid == 0) s_odd = 0;
    int t_begin = wg_lo / KT, t_end = wg_hi > 0 ? (wg_hi + KT - 1) / KT : 0;
    t_begin = min(t_begin, t_end);   // no key at all: no tile
    if (p.splits > 1) {
        const int per = (int) div31((unsigned) (t_end - t_begin + p.splits - 1), p.by_splits);
        t_begin = min(t_end, t_begin + split * per);
        t_end = min(t_end, t_begin + per);
    }

    // staging: load i of a wavefront takes the rows (wave LOADS + i) ROWS + lane / UNITS of a tile, 16 bytes a lane
    const char *kb = reinterpret_cast<const char *>(p.k + b * p.ks[0] + kvh * p.ks[1]), *vb = reinterpret_cast<const char *>(p.v + b * p.vs[0] + kvh * p.vs[1]);
    const unsigned k_step = (unsigned) p.ks[2] * 2u, v_step = (unsigned) p.vs[2] * 2u;
    const int s_row = wave * LOADS * ROWS + lane / UNITS, s_unit = lane % UNITS;
    u32x4 k_reg[LOADS], v_reg[LOADS];
    auto fetch = [&](int t) __attribute__((always_inline)) {   // rows past the last key come as zeros
        const int left = min(p.k_tokens - t * KT, KT);
        const rsrc_t rk = make_rsrc(kb + (long long) t * KT * k_step, (unsigned) (left - 1) * k_step + HD * 2u);
        const rsrc_t rv = make_rsrc(vb + (long long) t * KT * v_step, (unsigned) (left - 1) * v_step + HD * 2u);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const unsigned row = (unsigned) (s_row + i * ROWS);
            k_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, row * k_step + s_unit * 16, 0, 0);
            v_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, row * v_step + s_unit * 16, 0, 0);
        }
    };
    // Where some row does not see all of a tile, an infinity or a NaN in v times its probability of zero is not zero: those values go into LDS as
    // zeros, and are added to the rows that see them behind the loop.
    unsigned odd = 0u;
    auto mixed = [&](int t) __attribute__((always_inline)) { return t * KT < wg_all_lo || t * KT + KT > wg_all_hi; };
    auto put = [&](int buf, bool clean) __attribute__((always_inline)) {
        if (clean) {   // uniform
            constexpr unsigned EXP = DT == DT_BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = EXP & ~(EXP << 1);   // the exponents, and one in each: the sum's top bits are their carries
            unsigned any = 0u;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) any |= (v_reg[i][j] & EXP) + ONE;
            if (__any((any & 0x80008000u) != 0u)) {
                odd = 1u;
#pragma unroll
                for (int i = 0; i < LOADS; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v_reg[i][j] = finite_of<DT>(v_reg[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = s_row + i * ROWS;
            *reinterpret_cast<u32x4 *>(s_kv + (buf * KT + row) * KP + s_unit * 16) = k_reg[i];
            *reinterpret_cast<u32x4 *>(Vs + (buf * KT + row) * VP + s_unit * 16) = v_reg[i];
        }
    };
    auto mfma = [](const uint4 &x, const uint4 &y, f32x16 c) __attribute__((always_inline)) {
        if constexpr (DT == DT_BF16)
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    };
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_t;
    // of 16 lanes, four read the 32 bytes of 16 channels of one key, and each gets four keys of one channel
    const int j16 = lane & 15;
    const unsigned char *const v_at = Vs + (4 * lh + j16 / 4) * VP + li / 16 * 32 + j16 % 4 * 8;
    auto v_frag = [&](int buf, int t, int g, int d) __attribute__((always_inline)) {   // keys 32 t + 16 g + 4 lh + .. and 8 + .. of channel tile d
        const unsigned char *at = v_at + buf * KT * VP + (32 * t + 16 * g) * VP + 64 * d;
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t) at));
        const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t) (at + 8 * VP)));
        return make_uint4(x.x, x.y, y.x, y.y);
    };

    if (t_begin < t_end) fetch(t_begin);
    // q on into the channels 16 s + 8 (lane / 32) .. + 7 of step s, through the wavefront's part of the second buffers (RG 8: of both)
    uint4 qf[STEPS];
    {
        unsigned char *const rows = RG == 8 ? s_kv + wave * 32 * KP : (wave < 2 ? s_kv + KT * KP : Vs + KT * VP) + (wave & 1) * 32 * KP;
#pragma unroll
        for (int i = 0; i < 32 / ROWS; ++i)
            *reinterpret_cast<u32x4 *>(rows + (i * ROWS + lane / UNITS) * KP + lane % UNITS * 16) = qr[i] ^ u32x4{p.flip, p.flip, p.flip, p.flip};
#pragma unroll
        for (int st = 0; st < STEPS; ++st) qf[st] = __builtin_bit_cast(uint4, *reinterpret_cast<const u32x4 *>(rows + li * KP + lh * 16 + st * 32));
    }
    if (RG == 8) __syncthreads();   // the first buffers were some wavefronts' parts
    f32x16 o[DTILES];
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    const float unit = HOW == GENERAL ? 1.0f : p.scale2;   // of the scores and of m, in units of the exponential base 2
    float m = -INFINITY, l = 0.0f;
    const float slope2 = HOW == GENERAL && p.slopes ? slope_within(p.slopes[head] * 1.44269504088896340736f) : 0.0f;
    // BIASED: keys' numbers in the channels 0 .. 2 and ones in 3 .. 5 times the parts of the quotient and of the rest
    const float ratio = HOW == BIASED ? slope_within(p.slopes[head] * p.per_scale) : 0.0f;
    uint4 numbers[NT], quotient = make_uint4(0u, 0u, 0u, 0u);
    auto parts_of = [](float x, unsigned (&part)[3]) __attribute__((always_inline)) {   // x as a sum of three bf16, in the upper halves
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            part[i] = __float_as_uint(x) & 0xffff0000u;
            x -= __uint_as_float(part[i]);
        }
    };
    if constexpr (HOW == BIASED) {
        unsigned part[3];
        parts_of(ratio, part);
        if (lh == 0) {
            quotient.x = part[0] >> 16 | part[1];
            quotient.y = part[2] >> 16;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const unsigned number = __float_as_uint((float) (32 * n + li)) >> 16;
            numbers[n] = make_uint4(number | number << 16, number | 0x3f800000u, 0x3f803f80u, 0u);   // times zeros in the lanes 32 ..
        }
    }

    auto tile = [&](int t, int buf) __attribute__((always_inline)) {
        const int key0 = t * KT + 32 * kh;   // the wavefront's part of the tile: 32 NT keys
        if (key0 >= any_hi || key0 + 32 * NT <= any_lo) return;   // uniform: none of the wavefront's rows sees it
        const bool whole = key0 >= all_lo && key0 + 32 * NT <= all_hi;
        // The order of a tile's instructions is kept as it stands here: operands AHEAD products before their use (the compiler, short of registers, asks for
        // each where it needs it)
        constexpr int AHEAD = 4;
        f32x16 s[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[n][r] = 0.0f;
        if constexpr (HOW == BIASED) {
            unsigned part[3];
            parts_of(lh == 0 ? ratio * (float) (key0 - place) : 0.0f, part);
            const uint4 by = make_uint4(quotient.x, quotient.y | part[0], part[1] >> 16 | part[2], 0u);
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, numbers[n]), __builtin_bit_cast(bf16x8, by), s[n], 0, 0, 0);
        }
        const unsigned char *const k_at = s_kv + (buf * KT + 32 * kh + li) * KP + lh * 16;
        auto k_frag = [&](int i) __attribute__((always_inline)) {
            return __builtin_bit_cast(uint4, *reinterpret_cast<const u32x4 *>(k_at + i / STEPS * 32 * KP + i % STEPS * 32));
        };
        uint4 ring[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ring[i] = k_frag(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NT * STEPS; ++i) {
            s[i / STEPS] = mfma(ring[i % AHEAD], qf[i % STEPS], s[i / STEPS]);
            if (i + AHEAD < NT * STEPS) ring[i % AHEAD] = k_frag(i + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (HOW == GENERAL) {
            if (p.cap.cap2 > 0.0f) {   // uniform
                float x[16 * NT];
#pragma unroll
                for (int i = 0; i < 16 * NT; ++i) x[i] = s[i / 16][i % 16];
                cap_scores(p.cap, x);
#pragma unroll
                for (int i = 0; i < 16 * NT; ++i) s[i / 16][i % 16] = x[i];
            }
            const float mul = p.cap.cap2 > 0.0f ? 1.0f : p.scale2;
            const float away = (float) (place - key0 - 4 * lh);   // of the lane's first key; the others follow at constant distances
            if (!p.slopes) {   // uniform
                if (!(p.cap.cap2 > 0.0f))
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[n][r] *= mul;
            } else if (p.causal) {   // the keys that count lie behind: the distance has no sign to lose
                const float base = -slope2 * away;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[n][r] = __builtin_fmaf(s[n][r], mul, __builtin_fmaf(slope2, (float) (32 * n + 8 * (r / 4) + r % 4), base));
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[n][r] = __builtin_fmaf(s[n][r], mul, -slope2 * fabsf(away - (float) (32 * n + 8 * (r / 4) + r % 4)));
            }
        }
        if (!whole) {   // the row's interval as bits of the lane's keys: two instructions a score
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int from = key0 + 32 * n + 4 * lh;
                auto below = [](int x) __attribute__((always_inline)) { return (1u << min(max(x, 0), 31)) - 1u; };   // bits up to 27 count
                const unsigned seen = below(hi - from) & ~below(lo - from);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const unsigned keep = (unsigned) ((int) (seen << (31 - (8 * (r / 4) + r % 4))) >> 31);
                    s[n][r] = __uint_as_float((__float_as_uint(s[n][r]) & keep) | (0xff800000u & ~keep));
                }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const bool far = top - m > p.far;   // (m + far would be rounded)  Each row by itself: its bits do not depend on the rows beside it
        if (__any(far)) {
            const float next = far ? top : m, fade = __builtin_amdgcn_exp2f((m - (next == -INFINITY ? 0.0f : next)) * unit);
            m = next;
            l *= fade;
#pragma unroll
            for (int d = 0; d < DTILES; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= fade;
        }
        float shift = m == -INFINITY ? 0.0f : __builtin_fmaf(-m, unit, SHIFT);
        if (__any(fabsf(shift) > 65536.0f)) {   // the sum would count the rounding of m: such rows' scores have m taken off first
            const bool high = fabsf(shift) > 65536.0f;
            const float from = high ? m : 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[n][r] -= from;
            shift = high ? SHIFT : shift;
        }
        constexpr int PRODUCTS = 2 * DTILES;   // of 32 keys
        auto v_ask = [&](int i) __attribute__((always_inline)) { return v_frag(buf, i / PRODUCTS + kh, i % PRODUCTS / DTILES, i % DTILES); };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ring[i] = v_ask(i);
        __builtin_amdgcn_sched_barrier(0);
        unsigned pk[NT][8];
        auto weigh = [&](int n, int j) __attribute__((always_inline)) {   // two probabilities
            const float x = __builtin_amdgcn_exp2f(HOW == GENERAL ? s[n][2 * j] + shift : __builtin_fmaf(s[n][2 * j], p.scale2, shift));
            const float y = __builtin_amdgcn_exp2f(HOW == GENERAL ? s[n][2 * j + 1] + shift : __builtin_fmaf(s[n][2 * j + 1], p.scale2, shift));
            pk[n][j] = pack_h16<DT>(x, y);
            // the sum is of the rounded ones: what rounding adds to all of a row's weights is divided out again
            if constexpr (DT == DT_BF16) l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pk[n][j]), bf16x2{(__bf16) 1.0f, (__bf16) 1.0f}, l, false);
            else l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pk[n][j]), f16x2{(_Float16) 1.0f, (_Float16) 1.0f}, l, false);
        };
#pragma unroll
        for (int j = 0; j < 8; ++j) weigh(0, j);
        __builtin_amdgcn_sched_barrier(0);
        // the second 32 keys' probabilities between the first ones' products
#pragma unroll
        for (int i = 0; i < NT * PRODUCTS; ++i) {
            const int n = i / PRODUCTS, g = i % PRODUCTS / DTILES, d = i % DTILES;
            o[d] = mfma(ring[i % AHEAD], make_uint4(pk[n][4 * g], pk[n][4 * g + 1], pk[n][4 * g + 2], pk[n][4 * g + 3]), o[d]);
            if (i + AHEAD < NT * PRODUCTS) ring[i % AHEAD] = v_ask(i + AHEAD);
            if (NT == 2 && n == 0)
#pragma unroll
                for (int j = 0; j < 8 / PRODUCTS; ++j) weigh(1, i * (8 / PRODUCTS) + j);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // of the two wavefronts that share a SIMD one goes first, so that its softmax is beside the other's products (4096 causal tokens of 32 heads 139 -> 135 us; the
    // second half a tile behind by a barrier between scores and values: 144)
    if (RG == 8 && wave < 4) __builtin_amdgcn_s_setprio(2);
    if (t_begin < t_end) {
        put(0, mixed(t_begin));
        if (t_begin + 1 < t_end) fetch(t_begin + 1);
        for (int t = t_begin; t < t_end; ++t) {
            const int buf = (t - t_begin) & 1;
            __syncthreads();   // tile t is in LDS, tile t - 1 has been read
            if (t + 1 < t_end) put(buf ^ 1, mixed(t + 1));
            if (t + 2 < t_end) fetch(t + 2);
            tile(t, buf);
        }
    }

    if (odd && lane == 0) s_odd = 1;
    __syncthreads();
    l += __shfl_xor(l, 32, 64);
    m *= unit;
    if constexpr (RG == 2) {   // the two halves of the keys: the second wavefront's results to the first
        float *const half = reinterpret_cast<float *>(s_kv) + rg * (DTILES * 16 + 2) * 64 + lane;
        static_assert(2 * (DTILES * 16 + 2) * 64 * 4 <= 2 * KT * KP, "two row groups, in the place of k");
        if (kh) {
            half[0] = m;
            half[64] = l;
#pragma unroll
            for (int d = 0; d < DTILES; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) half[(2 + d * 16 + r) * 64] = o[d][r];
        }
        __syncthreads();
        if (!kh) {
            const float other = half[0], next = fmaxf(m, other), ref = next == -INFINITY ? 0.0f : next;
            const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(other - ref);
            m = next;
            l = l * f0 + half[64] * f1;
#pragma unroll
            for (int d = 0; d < DTILES; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * f0 + half[(2 + d * 16 + r) * 64] * f1;
        }
    }
    if (s_odd) {   // uniform and rare: for infinities of either sign and NaN, how many of a channel a row sees
        constexpr unsigned ONE = DT == DT_BF16 ? 0x3f80u : 0x3c00u;
        const unsigned span = (unsigned) (hi - lo);
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll 1
            for (int what = 0; what < 3; ++what) {
                f32x16 z;
#pragma unroll
                for (int r = 0; r < 16; ++r) z[r] = 0.0f;
#pragma unroll 1
                for (int t = t_begin; t < t_end; ++t) {
                    if (!mixed(t)) continue;   // uniform in the workgroup
                    __syncthreads();
                    fetch(t);
                    put(0, false);
                    __syncthreads();
#pragma unroll 1
                    for (int i = 0; i < KT / 16; ++i) {
                        unsigned seen[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = t * KT + 16 * i + 8 * (j / 2) + 4 * lh + j % 2 * 2;
                            seen[j] = ((unsigned) (key - lo) < span ? ONE : 0u) | ((unsigned) (key + 1 - lo) < span ? ONE << 16 : 0u);
                        }
                        const uint4 x = v_frag(0, 0, i, d);
                        z = mfma(make_uint4(special_of<DT>(x.x, what), special_of<DT>(x.y, what), special_of<DT>(x.z, what), special_of<DT>(x.w, what)),
                                 make_uint4(seen[0], seen[1], seen[2], seen[3]), z);
                    }
                }
                const float value = what == 0 ? INFINITY : what == 1 ? -INFINITY : NAN;
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] += z[r] > 0.0f ? value : 0.0f;
            }
        __syncthreads();
    }

    if (kh) return;
    if (m == -INFINITY && l == 0.0f && lo < hi) l = p.splits > 1 ? 1.0f : NAN;   // the row sees keys, and every score is minus infinity: no number, unless another part has one
    if (p.splits > 1) {
        unsigned again = row0;   // the row's token and head anew, not kept through the loop
        asm volatile("" : "+s"(again));
        again += (unsigned) li;
        if (again > last_row) return;
        token = (int) div31(again, p.by_group);
        head = kvh * p.group + (int) (again - (unsigned) token * (unsigned) p.group);
        const long long row = ((long long) b * p.q_heads + head) * p.q_tokens + token;
        if (lh == 0) *reinterpret_cast<float2 *>(p.part_ml + (row * p.splits + split) * 2) = make_float2(m, l);
        if (t_begin >= t_end) return;
        float *po = p.part_o + (row * p.splits + split) * HD;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4 *>(po + 32 * d + 8 * g + 4 * lh) = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
        return;
    }
    // the result as q came, through LDS: whole rows to memory (in the place of k, or of v where the halves of the keys are joined in that)
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    unsigned char *const rows = (RG >= 4 ? s_kv : Vs) + rg * 32 * KP;
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2 *>(rows + li * KP + 64 * d + 16 * g + 8 * lh) =
                make_uint2(pack_h16<DT>(o[d][4 * g] * inv, o[d][4 * g + 1] * inv), pack_h16<DT>(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
#pragma unroll
    for (int i = 0; i < 32 / ROWS; ++i) {
        const unsigned row = row0 + (unsigned) (i * ROWS + lane / UNITS), tk = div31(min(row, last_row), p.by_group);
        const u32x4 x = *reinterpret_cast<const u32x4 *>(rows + (i * ROWS + lane / UNITS) * KP + lane % UNITS * 16);
        if (row <= last_row)
            *reinterpret_cast<u32x4 *>(p.out + b * p.os[0] + (long long) (kvh * p.group + (int) (row - tk * (unsigned) p.group)) * p.os[1] + tk * p.os[2] + lane % UNITS * 8) = x;
    }
}

// Rows of a workgroup (32 rg), and parts of the keys where row blocks alone leave compute units without work.
//   256 rows, for which a tile is staged half as often, with head dimension 128: where workgroups, one a compute unit, fill seven eighths of two rounds or more and
//     blocks are no more than a sixteenth larger than the rows (4096 causal tokens of 32 heads 162 -> 141 us, 4096 on 16384 keys 970 -> 873; 2560 tokens, 320
//     workgroups in 512 places, 74 and 77, 16 x 260 of 32 heads on 32 46 and 59; 8192 of 16 heads of 64, whose registers give way, 182 and 214); and where as many
//     parts as fill one round have 640 keys of the middle row each, two parts 1600 (the last 512 of 8000 tokens of 32 heads on 8 126 -> 79 us, of 16000 245 -> 137, 256 of
//     6000 47 -> 41, 768 of 8000 162 -> 123; 1000 of 3000 62 and 66).
//   64 rows where 128 give no more than one workgroup a compute unit (4096 causal tokens of 8 heads on one 91 -> 72 us, 2048 of 16 heads of 64 34.5 -> 27, 77 of 12
//     7.0 -> 6.0); above that they stage every tile twice as often (2048 of 32 heads 56 and 66 us).  In parts of 256 keys at least where those do not give one
//     a compute unit either (one token of 32 heads on 4096 keys 13.5 us, with 512 keys a part 17).
static void masked_shape(const onhip_masked_attention_desc_t *d, int *rg, long long *blocks, int *splits) {
    const long long total = (long long) d->q_tokens * (d->q_heads / d->kv_heads), pairs = (long long) d->batch * d->kv_heads;
    const long long wide = (total + 255) / 256, items = wide * pairs, rounds = (items + 255) / 256;
    long long keys = d->k_tokens, parts = 1;
    if (d->window > 0 && d->window + 128LL < keys) keys = d->window + 128LL;
    const long long middle = d->causal ? (long long) d->q_offset + d->q_tokens / 2 : keys, seen = middle < 0 ? 0 : middle < keys ? middle : keys;   // by the middle row
    if ((total + 127) / 128 * pairs > 256) {
        *rg = d->head_dim == 128 && rounds > 1 && wide * 256 <= total + total / 16 && items * 8 >= rounds * 256 * 7 ? 8 : 4;
    } else if (d->head_dim == 128 && items <= 128 && wide * 256 <= 2 * total && seen / (256 / items) >= (items <= 85 ? 640 : 1600)) {
        *rg = 8;
        parts = 256 / items;
    } else {
        *rg = 2;
        const long long all = (total + 63) / 64 * pairs, most = (keys + 255) / 256;
        if (all < 256) parts = (512 + all - 1) / all < most ? (512 + all - 1) / all : most;
    }
    *blocks = (total + 32 * *rg - 1) / (32 * *rg);
    *splits = parts < 1 ? 1 : parts > 256 ? 256 : (int) parts;
}

static int masked_check(const onhip_masked_attention_desc_t *d, int *dt, int *rg, int *blocks, int *splits) {
    constexpr int MOST = 1 << 29;
    if (!d || d->batch < 1 || d->q_heads < 1 || d->kv_heads < 1 || d->q_tokens < 1 || d->k_tokens < 0) return set_error(ONHIP_ERR_ARG, "masked attention: bad shape");
    if (d->compute == ONHIP_COMPUTE_BF16) *dt = DT_BF16;
    else if (d->compute == ONHIP_COMPUTE_F16) *dt = DT_F16;
    else return set_error(ONHIP_ERR_ARG, "masked attention: compute type %d is neither bf16 nor fp16", d->compute);
    if (d->head_dim != 64 && d->head_dim != 128) return set_error(ONHIP_ERR_ARG, "masked attention: head dimension %d (64 and 128 are available)", d->head_dim);
    if (d->q_heads % d->kv_heads) return set_error(ONHIP_ERR_ARG, "masked attention: %d query heads for %d key-value heads", d->q_heads, d->kv_heads);
    if (d->k_tokens > MOST || d->q_tokens > MOST || d->q_offset > MOST || d->q_offset < -MOST) return set_error(ONHIP_ERR_ARG, "masked attention: lengths and places are at most 2^29");
    if (d->window < 0 || d->window > MOST) return set_error(ONHIP_ERR_ARG, "masked attention: a window of %d", d->window);
    if (!cap_fits(d->scale, d->softcap)) return set_error(ONHIP_ERR_ARG, "masked attention: scale and cap must be below 10^30 and finite, the cap not negative, their quotient between 10^-30 and 10^30");
    const long long heads = (long long) d->batch * d->q_heads;
    if (heads >= (1LL << 31) || heads * d->q_tokens >= (1LL << 31)) return set_error(ONHIP_ERR_ARG, "masked attention: too many rows");
    long long n;
    masked_shape(d, rg, &n, splits);
    if (n * d->batch * d->kv_heads >= (1LL << 22)) return set_error(ONHIP_ERR_ARG, "masked attention: too many rows");
    *blocks = (int) n;
    return ONHIP_OK;
}

template <int DT, int HD, int HOW>
static int masked_launch(const MaskedParams &p, int rg, hipStream_t stream) {
    const dim3 grid((unsigned) p.batch * p.kv_heads * p.blocks * p.splits);
    if constexpr (HD == 128)
        if (rg == 8) {
            hipLaunchKernelGGL((attention_masked_kernel<DT, HD, HOW, 8>), grid, dim3(512), 0, stream, p);
            ONHIP_CHECK_HIP(hipGetLastError());
            return ONHIP_OK;
        }
    if (rg == 2) hipLaunchKernelGGL((attention_masked_kernel<DT, HD, HOW, 2>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((attention_masked_kernel<DT, HD, HOW, 4>), grid, dim3(256), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

}  // namespace onhip

using namespace onhip;

extern "C" {

size_t onhip_attention_masked_workspace(const onhip_masked_attention_desc_t *d) {
    int dt, rg, blocks, splits;
    if (masked_check(d, &dt, &rg, &blocks, &splits)) return 0;
    return join_bytes((long long) d->batch * d->q_heads * d->q_tokens, splits, d->head_dim);
}

int onhip_attention_masked(const onhip_masked_attention_desc_t *d, const void *q, const void *k, const void *v, const int32_t *ranges,
                           const float *slopes, void *out, void *workspace, size_t workspace_bytes, void *stream) {
    MaskedParams p;
    int dt, rg;
    const int rc = masked_check(d, &dt, &rg, &p.blocks, &p.splits);
    if (rc) return rc;
    if (!q || !out || (d->k_tokens > 0 && (!k || !v))) return set_error(ONHIP_ERR_ARG, "masked attention: null tensor pointer");
    if (out == q || (d->k_tokens > 0 && (out == k || out == v))) return set_error(ONHIP_ERR_ARG, "masked attention: the result may not be an operand");
    if (reinterpret_cast<uintptr_t>(ranges) % 8) return set_error(ONHIP_ERR_ARG, "masked attention: ranges must be 8-byte aligned");
    const long long *strides[4] = {d->q_strides, d->k_strides, d->v_strides, d->out_strides};
    const void *ptrs[4] = {q, k, v, out};
    const int q_extent[3] = {d->batch, d->q_heads, d->q_tokens}, k_extent[3] = {d->batch, d->kv_heads, d->k_tokens};
    long long *const own[4] = {p.qs, p.ks, p.vs, p.os};
    for (int t = 0; t < 4; ++t) {
        const bool of_k = t == 1 || t == 2;
        if (reinterpret_cast<uintptr_t>(ptrs[t]) % 16) return set_error(ONHIP_ERR_ARG, "masked attention: tensors must be 16-byte aligned");
        for (int i = 0; i < 3; ++i) {
            own[t][i] = 0;   // a stride that is never stepped over
            if ((of_k ? k_extent : q_extent)[i] <= 1) continue;
            if (strides[t][i] < 0 || strides[t][i] % 8) return set_error(ONHIP_ERR_ARG, "masked attention: strides must be non-negative multiples of 8");
            own[t][i] = strides[t][i];
        }
    }
    if (!rows_apart(q_extent, d->out_strides, d->head_dim)) return set_error(ONHIP_ERR_ARG, "masked attention: rows of the result overlap");
    if (p.ks[2] >= (1LL << 23) || p.vs[2] >= (1LL << 23)) return set_error(ONHIP_ERR_ARG, "masked attention: token strides of k and v must be below 2^23");
    const long long rows = (long long) d->batch * d->q_heads * d->q_tokens;
    const size_t need = join_bytes(rows, p.splits, d->head_dim);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(ONHIP_ERR_WORKSPACE, "masked attention: a 16-byte aligned workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t) 0);
    p.q = reinterpret_cast<const unsigned short *>(q);
    p.k = reinterpret_cast<const unsigned short *>(k);
    p.v = reinterpret_cast<const unsigned short *>(v);
    p.out = reinterpret_cast<unsigned short *>(out);
    p.ranges = ranges;
    p.slopes = slopes;
    p.batch = d->batch;
    p.q_heads = d->q_heads;
    p.kv_heads = d->kv_heads;
    p.group = d->q_heads / d->kv_heads;
    p.q_tokens = d->q_tokens;
    p.k_tokens = d->k_tokens;
    p.q_offset = d->q_offset;
    p.causal = d->causal;
    p.window = d->window;
    p.spread = (long long) d->batch * d->kv_heads % 8 == 0;
    p.by_splits = make_div31((unsigned) p.splits);
    p.by_heads = make_div31((unsigned) (d->batch * d->kv_heads) / (p.spread ? 8u : 1u));
    p.by_kv_heads = make_div31((unsigned) d->kv_heads);
    p.by_group = make_div31((unsigned) p.group);
    p.flip = d->scale < 0.0f ? 0x80008000u : 0u;
    p.scale2 = fabsf(d->scale) * 1.44269504088896340736f;
    p.cap = make_cap(fabsf(d->scale), d->softcap);
    p.part_o = reinterpret_cast<float *>(workspace);
    p.part_ml = p.part_o + rows * p.splits * d->head_dim;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool usual = d->softcap == 0.0f && fabsf(d->scale) >= 1e-6f;   // a quotient of slope and scale stays in fp32's range
    p.per_scale = usual ? 1.0f / fabsf(d->scale) : 0.0f;
    p.far = usual && (!slopes || d->causal) ? 8.0f / p.scale2 : 8.0f;
    auto by_how = [&]<int DT, int HD>() {
        if (usual && !slopes) return masked_launch<DT, HD, PLAIN>(p, rg, st);
        return usual && d->causal ? masked_launch<DT, HD, BIASED>(p, rg, st) : masked_launch<DT, HD, GENERAL>(p, rg, st);
    };
    auto by_size = [&]<int DT>() { return d->head_dim == 64 ? by_how.template operator()<DT, 64>() : by_how.template operator()<DT, 128>(); };
    const int done = dt == DT_BF16 ? by_size.template operator()<DT_BF16>() : by_size.template operator()<DT_F16>();
    if (done || p.splits == 1) return done;
    JoinParams j;
    j.o = p.part_o;
    j.ml = p.part_ml;
    j.out = p.out;
    for (int i = 0; i < 3; ++i) j.os[i] = p.os[i];
    j.heads = p.q_heads;
    j.tokens = p.q_tokens;
    j.splits = p.splits;
    j.rows = rows;
    return attention_join_launch(dt, d->head_dim, j, st);
}

}  // extern "C"
