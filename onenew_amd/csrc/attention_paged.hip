// Attention of one new token a sequence over a paged key-value cache:  s_j = cap tanh(scale q.k_j / cap) - slope (len - 1 - j),  out = Softmax(s) v
// over the keys j of [max(0, len - window), len), in one pass over the cache with the running maximum and sum of a softmax.
//
// Up to 16 query heads that share a key-value head are the columns of the matrix instructions (v_mfma_f32_16x16x32), so the cache is read
// once for all of them.  A wavefront takes tiles of 32 keys by itself, with no barrier until its end: S^T = K q^T, whose result leaves a
// lane with a quarter of the scores of one head; and out^T = V^T P^T, whose second operand is those scores' exponentials where they are.  Both operands of
// the cache are read whole rows at a time, 4 to 16 lanes a row.  K turns into operands through the wavefront's own part of LDS (straight into them,
// a row a lane, cost 64 cycles of a compute unit's address path a load: 2.1 us for 128 KB, and 0.9 now).  V needs no such turn: a lane has the channels 8 li .. + 7
// (HD 128) of 8 keys, and channel 8 li + t of them is its operand for channel tile t, put together from the halves (or bytes) of those registers.
//
// Bound by memory: a byte of the cache takes part in 2 to 16 operations.  Measured against a large copy's 5.1 TB/s: 32 sequences of 2048 to 4096 keys, 8
// key-value heads of 128 in bf16, 407 MB in 76 to 80 us; 4 of up to 65536 in int8 450 MB in 91 to 94 us; one of 65536 in bf16 268 MB in 55 us; one of 777 10 us, its chain of
// trips to memory.  Workgroups a compute unit: two with head dimension 64 and int8 (128 registers), one else (16-bit rows of 64 channels 132 registers, four past two).  A sequence's tiles are shared out among `splits` workgroups of eight wavefronts, whose parts a second launch joins, where
// (sequence, head) pairs alone would leave compute units idle.
//
// int8: an int8 is a bf16 and an fp16, so the products are exact in it; the scale of a key multiplies its score, the scale of a value its
// probability.  Before the second product 2^(s - m) (times a constant) is rounded to fp16 with fp16 values, half of one of its eleven bits, and what is summed is the
// rounded one; with bf16 values, and with int8's times the scale, it goes in as two bf16 parts, sixteen bits: the cache's trip leaves the matrix cores time for both.
// (int8 in fp16, which has not the range for scales, needs a unit for them: in units of the largest one so far, one of 10^9 times the others took their
// bits although its key had no weight.)  Scores, maximum, sum and products' sums are fp32.
#include "attention_join.hpp"
#include "kv_common.hpp"

namespace onhip {

struct PagedParams {
    CacheView c;
    const unsigned short *q;
    unsigned short *out;
    long long qs[2], os[2];      // elements: (sequence, head)
    const int *table, *lengths;
    const float *slopes;
    long long table_stride;
    int table_pages, batch, q_heads, kv_heads, group, head_blocks, splits, window;
    float scale2;                // scale * log2(e)
    Cap cap;
    float *part_o, *part_ml;
};

constexpr float LOG2E = 1.44269504088896340736f;

// SMALL: pages of fewer than 16 tokens (a tile then has a page a lane; else two pages, the same for all lanes)
template <int DT, int HD, bool I8, bool SMALL>
__global__ __launch_bounds__(512, 2) void attention_paged_kernel(const PagedParams p) {
    constexpr int TILES = HD / 16, STEPS = HD / 32, NW = 8;
    constexpr int UNITS = (I8 ? 1 : 2) * HD / 16;     // 16-byte units of a key: 4, 8 or 16 lanes take one
    constexpr int KT = 32, NS = 8;                    // keys of a tile, scores of a lane
    constexpr int ROWS = 64 / UNITS, KW = KT / ROWS;  // keys of a load, loads of a tile
    constexpr int VB = (I8 ? 1 : 2) * HD / 16;        // bytes of a lane's part of a value: 4, 8 or 16
    constexpr int VW = VB / 4;
    // probabilities are 2^(s - m + SHIFT): fp16's stay clear of its smallest numbers, a sum of bf16's largest values of fp32's largest
    // (values below 2^-94, which are 2^-118 there, lose bits)
    constexpr int PT = I8 ? DT_BF16 : DT;   // type of the second product: a probability times a value's scale needs fp32's range
    constexpr float SHIFT = PT == DT_BF16 ? -24.0f : 7.0f;
    // a wavefront's tile of keys on its way into operands, in the end the wavefronts' results
    constexpr int KEY_BYTES = NW * KT * UNITS * 16, OUT_BYTES = NW * 16 * (HD + 4) * 4;
    __shared__ __attribute__((aligned(16))) unsigned char s_mem[KEY_BYTES > OUT_BYTES ? KEY_BYTES : OUT_BYTES];
    __shared__ float s_m[NW][16], s_l[NW][16];
    float(*s_o)[16][HD + 4] = reinterpret_cast<float(*)[16][HD + 4]>(s_mem);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;
    unsigned id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int hb = id % p.head_blocks;
    id /= p.head_blocks;
    const int kvh = id % p.kv_heads, b = id / p.kv_heads;

    const int reach = p.lengths[b];
    const long long room = (long long) p.table_pages << p.c.page_shift;
    const bool too_long = reach > room;   // more tokens than the table has pages for: the result is NaN
    const int len = too_long ? (int) room : reach;
    const int begin = p.window > 0 && len > p.window ? len - p.window : 0;
    const int tile0 = begin / KT, tiles = len > 0 ? (len + KT - 1) / KT - tile0 : 0;
    // as many parts as there are, each with a tile for every wavefront
    const int parts = min(p.splits, (tiles + NW - 1) / NW), per = parts > 0 ? (tiles + parts - 1) / parts : 0;
    const int t_begin = tile0 + split * per, t_end = min(t_begin + per, tile0 + tiles);

    const int head = hb * 16 + li;
    const bool live = head < p.group;
    const int qh = kvh * p.group + head;
    uint4 qf[STEPS];
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
        qf[st] = make_uint4(0u, 0u, 0u, 0u);
        // the channels that this lane's part of a key has in step st
        const int d = I8 ? st / 2 * 64 + lg * 16 + st % 2 * 8 : st * 32 + lg * 8;
        if (live) qf[st] = *reinterpret_cast<const uint4 *>(p.q + b * p.qs[0] + qh * p.qs[1] + d);
    }
    const float slope2 = p.slopes && live ? slope_within(p.slopes[qh] * LOG2E) : 0.0f;

    auto mfma = []<int T>(const uint4 &x, const uint4 &y, f32x4 c) __attribute__((always_inline)) {
        if constexpr (T == DT_BF16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    };

    f32x4 o[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    bool bad = false;
    const int *table = p.table + b * p.table_stride;
    const char *kb = p.c.k + kvh * p.c.ks[1], *vb = p.c.v + kvh * p.c.vs[1];

    const unsigned k_lane = (unsigned) (lane / UNITS) * (unsigned) p.c.ks[2] + lane % UNITS * 16, v_lane = 4u * lg * (unsigned) p.c.vs[2] + li * VB;
    u32x4 *const mine = reinterpret_cast<u32x4 *>(s_mem) + wave * KT * UNITS;
    auto unit_at = [](int row, int u) { return row * UNITS + (u ^ (row / (16 / UNITS) & (UNITS - 1))); };   // 16 lanes that take one unit of 16 keys meet every bank once

    // A tile as it is in flight: while one is worked on, the wavefront's next one is on its way, and the pages of the one behind that.
    struct Tile {
        u32x4 kr[KW];
        unsigned vf[NS][VW];
        float k_scale, v_scale;   // of key `lane` of the tile
    };
    struct Pages {   // of the tile's sixteens of keys, or of key `lane`
        int at[SMALL ? 1 : 2];
    };
    auto find = [&](int t, Pages &g) __attribute__((always_inline)) {
        const int key0 = t * KT;
        if constexpr (SMALL) {
            const int key = key0 + (lane & (KT - 1));
            g.at[0] = key >= begin && key < len ? table[key >> p.c.page_shift] : 0;
        } else {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int key = key0 + 16 * a;
                g.at[a] = key + 16 > begin && key < len ? table[key >> p.c.page_shift] : 0;
            }
        }
    };
    auto load = [&](int t, const Pages &g, Tile &x) __attribute__((always_inline)) {
        const int key0 = t * KT;
        int pg[2];
        if constexpr (SMALL) {
            const bool none = (unsigned) g.at[0] >= (unsigned) p.c.pages;
            bad |= none;
            pg[0] = none ? 0 : g.at[0];
        } else {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const bool none = (unsigned) g.at[a] >= (unsigned) p.c.pages;
                bad |= none;
                pg[a] = __builtin_amdgcn_readfirstlane(none ? 0 : g.at[a]);
            }
        }
        auto page_of = [&](int in_tile) __attribute__((always_inline)) { return __shfl(pg[0], in_tile, 64); };   // of key key0 + in_tile
        // what lies outside [begin, len) is read as well, from rows of pages that exist, and left out of the work.  Sixteen keys of a page: a
        // uniform address and the lane's own offset.
        const char *half_k[2], *half_v[2];
        if constexpr (!SMALL)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                half_k[a] = kb + pg[a] * p.c.ks[0] + ((key0 + 16 * a) & p.c.page_mask) * p.c.ks[2];
                half_v[a] = vb + pg[a] * p.c.vs[0] + ((key0 + 16 * a) & p.c.page_mask) * p.c.vs[2];
            }
#pragma unroll
        for (int i = 0; i < KW; ++i) {
            const char *src;
            if constexpr (SMALL) {
                const int row = i * ROWS + lane / UNITS;
                src = kb + page_of(row) * p.c.ks[0] + ((key0 + row) & p.c.page_mask) * (int) p.c.ks[2] + lane % UNITS * 16;
            } else {
                src = half_k[i * ROWS / 16] + (i * ROWS % 16) * p.c.ks[2] + k_lane;
            }
            x.kr[i] = *reinterpret_cast<const u32x4 *>(src);
        }
        if constexpr (I8) {
            const int page = SMALL || lane % 32 < 16 ? pg[0] : pg[1];
            const long long at = page * p.c.ss[0] + kvh * p.c.ss[1] + ((key0 + (lane & (KT - 1))) & p.c.page_mask) * p.c.ss[2];
            x.k_scale = p.c.k_scale[at];
            x.v_scale = p.c.v_scale[at];
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            const char *src;
            if constexpr (SMALL) {
                const int at = 16 * (j / 4) + 4 * lg + j % 4;
                src = vb + page_of(at) * p.c.vs[0] + ((key0 + at) & p.c.page_mask) * (int) p.c.vs[2] + li * VB;
            } else {
                src = half_v[j / 4] + (j % 4) * p.c.vs[2] + v_lane;
            }
            if constexpr (VB == 16) {
                const uint4 y = *reinterpret_cast<const uint4 *>(src);
                x.vf[j][0] = y.x; x.vf[j][1] = y.y; x.vf[j][2] = y.z; x.vf[j][3] = y.w;
            } else if constexpr (VB == 8) {
                const uint2 y = *reinterpret_cast<const uint2 *>(src);
                x.vf[j][0] = y.x; x.vf[j][1] = y.y;
            } else {
                x.vf[j][0] = *reinterpret_cast<const unsigned *>(src);
            }
        }
    };
    auto work = [&](int t, Tile &tile) __attribute__((always_inline)) {
        const int key0 = t * KT;
        const bool whole = key0 >= begin && key0 + KT <= len;   // uniform
        auto &vf = tile.vf;
#pragma unroll
        for (int i = 0; i < KW; ++i) mine[unit_at(i * ROWS + lane / UNITS, lane % UNITS)] = tile.kr[i];
        float ksc[NS], vsc[NS];
        if constexpr (I8) {
            const int key = key0 + (lane & (KT - 1));
            const bool seen = key >= begin && key < len;
            const float x = seen ? tile.k_scale : 0.0f;
            const float y = seen ? tile.v_scale : 0.0f;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int from_lane = 16 * (j / 4) + 4 * lg + j % 4;
                ksc[j] = __shfl(x * (p.cap.cap2 > 0.0f ? 1.0f : p.scale2), from_lane, 64);
                vsc[j] = __shfl(y, from_lane, 64);
            }
        }
        if (!whole) {   // a value that is not seen may be an infinity, and 0 of it is not 0
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int key = key0 + 16 * (j / 4) + 4 * lg + j % 4;
#pragma unroll
                for (int i = 0; i < VW; ++i) vf[j][i] = key >= begin && key < len ? vf[j][i] : 0u;
            }
        }

        // S^T: this lane's scores are of head li and the keys 16 (j / 4) + 4 lg + j % 4
        float s[NS];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (I8) {
                u32x4 x;
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    if (st % 2 == 0) x = mine[unit_at(16 * a + li, st * 2 + lg)];
                    const unsigned two[2] = {st % 2 ? x.z : x.x, st % 2 ? x.w : x.y};
                    unsigned y[4];
                    s8_to_h16<DT>(two, y);
                    acc = mfma.template operator()<DT>(make_uint4(y[0], y[1], y[2], y[3]), qf[st], acc);
                }
            } else {
#pragma unroll
                for (int st = 0; st < STEPS; ++st) acc = mfma.template operator()<DT>(__builtin_bit_cast(uint4, mine[unit_at(16 * a + li, st * 4 + lg)]), qf[st], acc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * a + r] = I8 ? acc[r] * ksc[4 * a + r] : acc[r];
        }
        if (p.cap.cap2 > 0.0f) {   // uniform
            cap_scores(p.cap, s);
        } else if constexpr (!I8) {
#pragma unroll
            for (int j = 0; j < NS; ++j) s[j] *= p.scale2;
        }
        if (p.slopes) {   // uniform
#pragma unroll
            for (int j = 0; j < NS; ++j) s[j] = __builtin_fmaf(slope2, (float) (key0 + 16 * (j / 4) + 4 * lg + j % 4 - (len - 1)), s[j]);
        }
        if (!whole) {
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int key = key0 + 16 * (j / 4) + 4 * lg + j % 4;
                if (key < begin || key >= len) s[j] = -INFINITY;
            }
        }
        float top = s[0];
#pragma unroll
        for (int j = 1; j < NS; ++j) top = fmaxf(top, s[j]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const bool far = top - m > 8.0f;   // the reference point follows a head's maximum when that is 2^8 above it: most tiles leave the sums alone
        if (__any(far)) {
            const float next = far ? top : m, fade = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.0f : next));
            m = next;
            l *= fade;
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[i][r] *= fade;
        }
        const float from = m == -INFINITY ? 0.0f : m;
        float e[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            e[j] = __builtin_amdgcn_exp2f(s[j] - from + SHIFT);   // SHIFT - m would be rounded
            if constexpr (PT == DT_BF16) l += e[j];
        }
        if constexpr (I8)
#pragma unroll
            for (int j = 0; j < NS; ++j) e[j] *= vsc[j];
        // out^T += V^T P^T: row i of channel tile n is the channel TILES i + n
        unsigned hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (PT == DT_BF16) {
                // a bf16 below the probability (or its size times a scale's), and the rest in a product of its own: of one sign both, so that an infinity stays one
                constexpr unsigned SIZE = I8 ? 0x7fffffffu : 0xffffffffu;   // a scale may have a sign
                const unsigned x = __float_as_uint(e[2 * i]), y = __float_as_uint(e[2 * i + 1]), x1 = x - ((x & SIZE) != 0u), y1 = y - ((y & SIZE) != 0u);
                hi[i] = __builtin_amdgcn_perm(y1, x1, 0x07060302u);
                lo[i] = pack_h16<PT>(e[2 * i] - __uint_as_float(x1 & 0xffff0000u), e[2 * i + 1] - __uint_as_float(y1 & 0xffff0000u));
            } else {
                hi[i] = pack_h16<PT>(e[2 * i], e[2 * i + 1]);
                lo[i] = 0u;
                // the sum is of the rounded ones: the weights of equal values sum to one
                l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, hi[i]), f16x2{(_Float16) 1.0f, (_Float16) 1.0f}, l, false);
            }
        }
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            unsigned a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (I8) {
                    const int x = (int) (vf[2 * i][n / 4] >> (n % 4 * 8)), y = (int) (vf[2 * i + 1][n / 4] >> (n % 4 * 8));
                    a[i] = pack_h16<PT>((float) (signed char) x, (float) (signed char) y);
                } else {
                    a[i] = __builtin_amdgcn_perm(vf[2 * i + 1][n / 2], vf[2 * i][n / 2], n % 2 ? 0x07060302u : 0x05040100u);
                }
            }
            const uint4 v4 = make_uint4(a[0], a[1], a[2], a[3]);
            o[n] = mfma.template operator()<PT>(v4, make_uint4(hi[0], hi[1], hi[2], hi[3]), o[n]);
            if constexpr (PT == DT_BF16) o[n] = mfma.template operator()<PT>(v4, make_uint4(lo[0], lo[1], lo[2], lo[3]), o[n]);
        }
    };

    int t = t_begin + wave;
    if (t < t_end) {
        Tile x, y;
        Pages now, next;
        const int last = t_end - 1;   // a tile asked for past the last one is the last one again, not worked on
        find(t, now);
        find(min(t + NW, last), next);
        load(t, now, x);
        for (;;) {
            find(min(t + 2 * NW, last), now);
            load(min(t + NW, last), next, y);
            work(t, x);
            t += NW;
            if (t >= t_end) break;
            find(min(t + 2 * NW, last), next);
            load(min(t + NW, last), now, x);
            work(t, y);
            t += NW;
            if (t >= t_end) break;
        }
    }
    // the eight wavefronts' parts
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (__any(bad) || too_long) l = NAN;
    if (lg == 0) {
        s_m[wave][li] = m;
        s_l[wave][li] = l;
    }
    __syncthreads();   // the last keys have been read
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < TILES; n += 4)
            *reinterpret_cast<float4 *>(&s_o[wave][li][(4 * lg + r) * TILES + n]) = make_float4(o[n][r], o[n + 1][r], o[n + 2][r], o[n + 3][r]);
    __syncthreads();
    constexpr int SHARE = 64 * NW / 16, PER = HD / SHARE;   // threads of a head, channels of a thread
    const int oh = threadIdx.x / SHARE, d0 = threadIdx.x % SHARE * PER;
    if (hb * 16 + oh >= p.group) return;
    float mm = s_m[0][oh];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, s_m[w][oh]);
    const float shift = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_m[w][oh] - shift);
        ll += s_l[w][oh] * f;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = __builtin_fmaf(s_o[w][oh][d0 + i], f, acc[i]);
        if (s_l[w][oh] != s_l[w][oh]) ll = NAN;   // a page that does not exist
    }
    if (mm == -INFINITY && ll == 0.0f && t_begin < t_end) ll = p.splits > 1 ? 1.0f : NAN;   // keys, and every score minus infinity: no number, unless another part has one
    const int row = b * p.q_heads + kvh * p.group + hb * 16 + oh;
    if (p.splits > 1) {
        float *po = p.part_o + ((long long) row * p.splits + split) * HD + d0;
#pragma unroll
        for (int i = 0; i < PER; i += 2) *reinterpret_cast<float2 *>(po + i) = make_float2(acc[i], acc[i + 1]);
        if (d0 == 0) *reinterpret_cast<float2 *>(p.part_ml + ((long long) row * p.splits + split) * 2) = make_float2(mm, ll);
        return;
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    unsigned short *dst = p.out + b * p.os[0] + (kvh * p.group + hb * 16 + oh) * p.os[1] + d0;
#pragma unroll
    for (int i = 0; i < PER; i += 2)
        reinterpret_cast<unsigned *>(dst)[i / 2] = pack_h16<DT>(acc[i] * inv, acc[i + 1] * inv);
}

// ---- the parts of a row joined ----------------------------------------------------------------------------------
// HD / 2 lanes of two channels take a part.  Few rows for their parts (SPREAD): all 8 or 16 groups of a workgroup on one row, joined through LDS, bound by its trips to memory: a
// group asks for eight parts at a time, the first eight before it knows their weights.  Many rows: a group has its own, bound by memory.
template <int DT, int HD, bool SPREAD>
__global__ __launch_bounds__(512) void attention_join_kernel(const JoinParams p) {
    constexpr int LANES = HD / 2, GROUPS = 512 / LANES, AHEAD = SPREAD ? 8 : 4, STEP = SPREAD ? GROUPS : 1;
    __shared__ float2 s_acc[SPREAD ? GROUPS : 1][LANES];
    __shared__ float s_l[GROUPS];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const long long row = SPREAD ? (long long) blockIdx.x : (long long) blockIdx.x * GROUPS + group;
    if (row >= p.rows) return;   // a whole group, and none that others wait for
    const float2 *ml = reinterpret_cast<const float2 *>(p.ml) + row * p.splits;
    const float2 *o = reinterpret_cast<const float2 *>(p.o + row * p.splits * HD) + lane;
    const int first = SPREAD ? group : 0;
    float2 part[AHEAD], own[AHEAD];
    auto ask = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = min(s0 + i * STEP, p.splits - 1);
            own[i] = ml[s];
            part[i] = o[(long long) s * LANES];
        }
    };
    ask(first);
    float mm = -INFINITY;
    for (int s = lane; s < p.splits; s += LANES) mm = fmaxf(mm, ml[s].x);
#pragma unroll
    for (int x = 1; x < LANES; x *= 2) mm = fmaxf(mm, __shfl_xor(mm, x, LANES));
    const float shift = mm == -INFINITY ? 0.0f : mm;
    float2 acc = make_float2(0.0f, 0.0f);
    float l = 0.0f;
    for (int s0 = first; s0 < p.splits; s0 += AHEAD * STEP) {
        if (s0 != first) ask(s0);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const bool there = s0 + i * STEP < p.splits, none = !there || own[i].x == -INFINITY;   // a part without keys has written no values
            const float f = none ? 0.0f : __builtin_amdgcn_exp2f(own[i].x - shift), ls = own[i].y;
            l += !none ? ls * f : there && (mm == -INFINITY ? ls != 0.0f : ls != ls) ? NAN : 0.0f;   // (a sum without a score: one of the row's keys, all of them minus infinity)
            acc.x = none ? acc.x : __builtin_fmaf(part[i].x, f, acc.x);   // a weight of 0 as well: what is no number stays
            acc.y = none ? acc.y : __builtin_fmaf(part[i].y, f, acc.y);
        }
    }
    if constexpr (SPREAD) {
        s_acc[group][lane] = acc;
        if (lane == 0) s_l[group] = l;
        __syncthreads();
        if (group) return;
        l = 0.0f;
        acc = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            l += s_l[g];
            acc.x += s_acc[g][lane].x;
            acc.y += s_acc[g][lane].y;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long token = row % p.tokens, bh = row / p.tokens, h = bh % p.heads, b = bh / p.heads;
    reinterpret_cast<unsigned *>(p.out + b * p.os[0] + h * p.os[1] + token * p.os[2])[lane] = pack_h16<DT>(acc.x * inv, acc.y * inv);
}

// (1024 rows in 64 parts spread 47 us of a call, not 51; in 16 parts 34 and 32.5; 16384 in 4 113 and 63)
template <int DT, int HD> static void join_launch(const JoinParams &p, hipStream_t stream) {
    constexpr int GROUPS = 1024 / HD;
    if (p.rows <= 16LL * p.splits) hipLaunchKernelGGL((attention_join_kernel<DT, HD, true>), dim3((unsigned) p.rows), dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((attention_join_kernel<DT, HD, false>), dim3((unsigned) ((p.rows + GROUPS - 1) / GROUPS)), dim3(512), 0, stream, p);
}

int attention_join_launch(int dt, int hd, const JoinParams &p, hipStream_t stream) {
    if (dt == DT_BF16) hd == 64 ? join_launch<DT_BF16, 64>(p, stream) : join_launch<DT_BF16, 128>(p, stream);
    else hd == 64 ? join_launch<DT_F16, 64>(p, stream) : join_launch<DT_F16, 128>(p, stream);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

// Workgroups that a sequence's head is cut into: as many that all of them are one a compute unit (two were 6 to 46 % behind: 32 sequences of 4096 keys 80 and 86 us, 2
// of 30000 with one key-value head 15.1 and 22.1), rounded up, and no more than the 256s of keys, rounded up as well (1025 keys: five parts of 205).  Where the heads do not divide
// 256, the rest is a second round of a few workgroups: of 4096 keys and eight heads 8 sequences take 25 us, 9 (288 workgroups) 33, 12 (288) 43, 17 (272) 56, 24 (384) 67, 32 78 and 33
// (264) 93.  Up to 1024 keys one, without a second launch (one sequence of 300 keys 7.3 us, in two parts
// 9.7; of 777 10.1 and in four 9.7, with a launch more to queue).  int8, whose tiles are half the bytes in flight: two a compute unit where each still has
// 4096 keys (4 of 65536 99 and 93 us; 32 of 4000 50 and 58).
static int paged_splits(const onhip_cache_desc_t *c, const onhip_paged_attention_desc_t *d) {
    const long long group = d->q_heads / c->kv_heads, rows = (long long) d->batch * c->kv_heads * ((group + 15) / 16);
    long long longest = (long long) d->table_pages * c->page_tokens;
    if (d->window > 0 && d->window < longest) longest = d->window;
    if (longest <= 1024) return 1;
    long long want = (256 + rows - 1) / rows;
    if (c->quantised && longest / (2 * want) >= 4096) want *= 2;
    const long long most = (longest + 255) / 256, s = want < most ? want : most;
    return s > 256 ? 256 : (int) s;
}

static int paged_check(const onhip_cache_desc_t *c, const onhip_paged_attention_desc_t *d, CacheView *view, int *dt) {
    const int rc = cache_shape("paged attention", c, view, dt);
    if (rc) return rc;
    if (!d || d->batch < 1 || d->q_heads < 1 || d->table_pages < 0 || d->table_stride < 0) return set_error(ONHIP_ERR_ARG, "paged attention: bad shape");
    if (d->q_heads % c->kv_heads) return set_error(ONHIP_ERR_ARG, "paged attention: %d query heads for %d key-value heads", d->q_heads, c->kv_heads);
    if ((long long) d->batch * d->q_heads >= (1LL << 22)) return set_error(ONHIP_ERR_ARG, "paged attention: %d sequences of %d heads", d->batch, d->q_heads);
    if ((long long) d->table_pages * c->page_tokens > (1LL << 30)) return set_error(ONHIP_ERR_ARG, "paged attention: a table of %d pages", d->table_pages);
    if (d->window < 0) return set_error(ONHIP_ERR_ARG, "paged attention: a window of %d", d->window);
    if (!cap_fits(d->scale, d->softcap)) return set_error(ONHIP_ERR_ARG, "paged attention: scale and cap must be below 10^30 and finite, the cap not negative, their quotient between 10^-30 and 10^30");
    return ONHIP_OK;
}

template <int DT, int HD, bool I8>
static int paged_launch(const PagedParams &p, unsigned blocks, hipStream_t stream) {
    if (p.c.page_shift < 4) hipLaunchKernelGGL((attention_paged_kernel<DT, HD, I8, true>), dim3(blocks), dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((attention_paged_kernel<DT, HD, I8, false>), dim3(blocks), dim3(512), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

}  // namespace onhip

using namespace onhip;

extern "C" {

size_t onhip_attention_paged_workspace(const onhip_cache_desc_t *c, const onhip_paged_attention_desc_t *d) {
    CacheView view;
    int dt;
    if (paged_check(c, d, &view, &dt)) return 0;
    return join_bytes((long long) d->batch * d->q_heads, paged_splits(c, d), c->head_dim);
}

int onhip_attention_paged(const onhip_cache_desc_t *c, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale,
                          const onhip_paged_attention_desc_t *d, const void *q, const int32_t *table, const int32_t *lengths,
                          const float *slopes, void *out, void *workspace, size_t workspace_bytes, void *stream) {
    PagedParams p;
    int dt, rc = paged_check(c, d, &p.c, &dt);
    if (!rc) rc = cache_memory("paged attention", c, k_cache, v_cache, k_scale, v_scale, &p.c);
    if (rc) return rc;
    if (!q || !out || !lengths || (d->table_pages > 0 && !table)) return set_error(ONHIP_ERR_ARG, "paged attention: null pointer");
    if (out == q) return set_error(ONHIP_ERR_ARG, "paged attention: the result may not be an operand");
    if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16) return set_error(ONHIP_ERR_ARG, "paged attention: tensors must be 16-byte aligned");
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = p.os[i] = 0;   // strides that are never stepped over
        if ((i == 0 ? d->batch : d->q_heads) == 1) continue;
        if (d->q_strides[i] < 0 || d->q_strides[i] % 8 || d->out_strides[i] < 0 || d->out_strides[i] % 8)
            return set_error(ONHIP_ERR_ARG, "paged attention: strides must be non-negative multiples of 8");
        p.qs[i] = d->q_strides[i];
        p.os[i] = d->out_strides[i];
    }
    const int extent[2] = {d->batch, d->q_heads};
    if (!rows_apart(extent, d->out_strides, c->head_dim)) return set_error(ONHIP_ERR_ARG, "paged attention: rows of the result overlap");
    if (out == k_cache || out == v_cache) return set_error(ONHIP_ERR_ARG, "paged attention: one memory for the result and the cache");
    const long long rows = (long long) d->batch * d->q_heads;
    p.splits = paged_splits(c, d);
    const size_t need = join_bytes(rows, p.splits, c->head_dim);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(ONHIP_ERR_WORKSPACE, "paged attention: a 16-byte aligned workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t) 0);
    p.q = reinterpret_cast<const unsigned short *>(q);
    p.out = reinterpret_cast<unsigned short *>(out);
    p.table = table;
    p.lengths = lengths;
    p.slopes = slopes;
    p.table_stride = d->table_stride;
    p.table_pages = d->table_pages;
    p.batch = d->batch;
    p.q_heads = d->q_heads;
    p.kv_heads = c->kv_heads;
    p.group = d->q_heads / c->kv_heads;
    p.head_blocks = (p.group + 15) / 16;
    p.window = d->window;
    p.scale2 = d->scale * LOG2E;
    p.cap = make_cap(d->scale, d->softcap);
    p.part_o = reinterpret_cast<float *>(workspace);
    p.part_ml = p.part_o + rows * p.splits * c->head_dim;
    const unsigned blocks = (unsigned) (d->batch * c->kv_heads * p.head_blocks * p.splits);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto by_size = [&]<int DT>() {
        if (c->head_dim == 64) return c->quantised ? paged_launch<DT, 64, true>(p, blocks, st) : paged_launch<DT, 64, false>(p, blocks, st);
        return c->quantised ? paged_launch<DT, 128, true>(p, blocks, st) : paged_launch<DT, 128, false>(p, blocks, st);
    };
    const int done = dt == DT_BF16 ? by_size.template operator()<DT_BF16>() : by_size.template operator()<DT_F16>();
    if (done || p.splits == 1) return done;
    JoinParams j;
    j.o = p.part_o;
    j.ml = p.part_ml;
    j.out = p.out;
    j.os[0] = p.os[0]; j.os[1] = p.os[1]; j.os[2] = 0;
    j.heads = p.q_heads;
    j.tokens = 1;
    j.splits = p.splits;
    j.rows = rows;
    return attention_join_launch(dt, c->head_dim, j, st);
}

}  // extern "C"
