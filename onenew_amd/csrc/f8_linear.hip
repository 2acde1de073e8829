// Product of rows and weights in 8-bit floating point:
//   out[m][n] = sum over blocks b of 128 channels  sa[m][b] sw[n / 128][b] (sum_k a[m][k] w[n][k])  + bias[n]
//
// A block's inner sums are matrix instructions that start at zero, sums over blocks fp32, a fused multiply-add a value.  Up to 32 rows, and for fp32 results, the instructions are those in bf16,
// which holds every e4m3: they wait for the weights there.  For 16-bit results of more rows they are those on e4m3 itself, in half the time: these add eight products at a time with 13 bits below the
// power of two of the largest one (what is below is cut), each eight joined in fp32.  Measured, root mean square: 2^-16 of the results' on random rows,
// 2^-14 where one channel of 128 is 300 times the others, of which single values can pass fp16's half step.  So a caller may ask for the sums of fp32 results (`exact`): 300 rows of 11008
// channels, 4096 outputs 45 instead of 38 us with weights from memory, 1024 rows of 4096 41 instead of 29, 8192 rows of 4096, 22016 outputs 1456 instead of 682.
// Weights are the instruction's rows, so that a lane's values belong to one row m and a lane has one factor a block and tile of sixteen rows, sa[m] times sw.
//
// Operands go from memory straight into LDS, a block of 128 channels of a row at a time; a row's 16-byte units are exchanged as (unit ^ row / 2 % 8), which puts the sixteen units that are
// read together on different banks.
//
// Three kernels: up to 32 rows a wavefront's own ring, bound by the weights' bytes; more rows tiles for a compute unit, bound by what goes into its LDS (48 to 56 bytes a cycle and unit are the
// most that direct loads reached); many rows tiles of 256 x 256, bound by matrix instructions and the multiply-adds of the scales beside them.
#include "f8_common.hpp"

namespace onhip {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct F8LinearParams {
    const char *a, *w;
    const float *a_scale, *w_scale, *bias;
    char *out;
    long long os;                    // bytes between rows
    int as, ws;
    long long a_ss[2], w_ss[2];      // floats between rows and blocks
    int m, n, k;
    int tiles_m, tiles_n;
    Div31 by_group, by_last;         // tiles in HIGH rows of them; rows of tiles in the last such group
    bool wide;                       // rows of results start at whole words
    bool quads;                      // scales of a row's blocks lie side by side, four of them at least
};

// a unit of 16 bytes of this lane from `voff` behind the descriptor's base (zeros outside) to LDS at `lds` + 16 lane.  In assembly, for the compiler waits for every
// such load in front of any LDS read; the waits are placed by hand.  Nothing else here goes by m0
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, unsigned voff, unsigned soff, unsigned lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" :: "s"(lds), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
#endif
}
// The units of a row that the four groups of sixteen lanes read, i = 0, 1: as both operands have the same, any order of the channels will do.  LDS reads 16 bytes of sixteen
// lanes at a time, of which eight are of one group and eight of another; units 0, 1, 6, 7 and 2, 3, 4, 5 keep those on different banks
__device__ __forceinline__ int lane_unit(int group, int i) { return i == 0 ? group + group / 2 * 4 : group + 2; }

// a word from each lane's address to LDS at `lds` + 4 lane
__device__ __forceinline__ void word_to_lds(const float *from, unsigned lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" :: "s"(lds), "v"(from) : "memory");
#endif
}
__device__ __forceinline__ void quad_to_lds(const float *from, unsigned lds) {   // four words, to `lds` + 16 lane
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds), "v"(from) : "memory");
#endif
}
__device__ __forceinline__ i32x4 f8_kept(i32x4 q, int keep) {   // the first `keep` of 16 bytes, the others zeros
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int bytes = keep - 4 * j;
        q[j] = bytes >= 4 ? q[j] : bytes <= 0 ? 0 : (int) ((unsigned) q[j] & (0xffffffffu >> (32 - 8 * bytes)));
    }
    return q;
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

// results n .. n + 3 of row m, as many as there are, with the bias
template <int DT> __device__ __forceinline__ void store4(const F8LinearParams &p, int m, int n, f32x4 v) {
    if (p.bias)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += n + j < p.n ? p.bias[n + j] : 0.0f;
    char *at = p.out + m * p.os + (long long) n * element_bytes<DT>;
    if (n + 4 <= p.n) {
        if constexpr (DT == DT_F32) *reinterpret_cast<any_f32x4 *>(at) = v;
        else *reinterpret_cast<any_u32x2 *>(at) = any_u32x2{pack_h16<DT>(v[0], v[1]), pack_h16<DT>(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < p.n) {
            if constexpr (DT == DT_F32) reinterpret_cast<float *>(at)[j] = v[j];
            else reinterpret_cast<unsigned short *>(at)[j] = (unsigned short) pack_h16<DT>(v[j], 0.0f);
        }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// A workgroup has 16 NT outputs of AM rows, its wavefronts a run of the blocks of channels each.  A wavefront has a place for a block in LDS of its own,
// which nobody else waits for, and takes the next one when it has read the last; whole lines come in (a load of matrix operands straight into registers takes sixteen rows at once, a line each:
// 10 bytes a cycle and compute unit were measured so).  The wavefronts' sums meet in LDS, in one order.  Deeper rings cost wavefronts a unit and were level or behind.
// Bound by the weights' bytes.  On the device, with weights from memory and from the last-level cache: 32 rows of 4096 channels, 22016 outputs 23.9 and 17.0 us (92 MB at 3.8 and 5.4 TB/s; a large
// copy reaches 4.9 to 5.4), 5 rows of 4000, 32003 fp32 outputs 28.4 and 21.5 us (129 MB, 4.5 and 6.0 TB/s); one row of 4096, 6144 outputs 7.5 and 4.9 us, where the launch and a wavefront's first
// loads count.
template <int DT, int AM, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void f8_few_kernel(const F8LinearParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int MT = AM < 16 ? 1 : AM / 16, CHUNK = 1024, SLOT = NT * 2048 + AM * 128 + 2 * CHUNK, RING = WAVES * SLOT, JOIN = WAVES * NT * MT * 1024;
    static_assert(AM < 64, "a lane for each row's scale, and for the weights'");
    __shared__ __attribute__((aligned(1024))) char lds[RING > JOIN ? RING : JOIN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lq = lane >> 4;
    const int n0 = (int) blockIdx.x * 16 * NT, m0 = (int) blockIdx.y * AM;
    const int k_blocks = (p.k + 127) / 128, k16 = (p.k + 15) & ~15, rows_n = min(16 * NT, p.n - n0), rows_m = min(AM, p.m - m0);
    const char *w_base = p.w + (long long) n0 * p.ws, *a_base = p.a + (long long) m0 * p.as;
    const unsigned w_bytes = (unsigned) ((rows_n - 1) * p.ws + k16), a_bytes = (unsigned) ((rows_m - 1) * p.as + k16);
    const int lrow = lane / 8;
    unsigned w_off[NT * 2], a_off[AM / 8];
#pragma unroll
    for (int t = 0; t < NT * 2; ++t) {
        const int row = t * 8 + lrow;
        w_off[t] = row < rows_n ? (unsigned) (row * p.ws) + ((lane % 8) ^ (row / 2 % 8)) * 16 : OOB;
    }
#pragma unroll
    for (int t = 0; t < AM / 8; ++t) {
        const int row = t * 8 + lrow;
        a_off[t] = row < rows_m ? (unsigned) (row * p.as) + ((lane % 8) ^ (row / 2 % 8)) * 16 : OOB;
    }
    // a lane's scale: of row `lane`, of the weights behind the rows
    const float *scales = lane < AM ? p.a_scale + (m0 + min(lane, rows_m - 1)) * p.a_ss[0] : p.w_scale + n0 / 128 * p.w_ss[0];
    const long long scale_step = lane < AM ? p.a_ss[1] : p.w_ss[1];
    const unsigned lds0 = (unsigned) (size_t) (__attribute__((address_space(3))) char *) lds + wave * SLOT;
    const i32x4 rw = descriptor(w_base, w_bytes), ra = descriptor(a_base, a_bytes);
    // a run of the blocks a wavefront; every WAVESth one where rows are not whole lines apart: two blocks then share a line, which wavefronts take at the same time (32003 outputs of
    // 4000 channels, 5 rows: 26.2 and 28.9 us; of 4096 channels 10% the other way)
    const bool spread = p.ws % 128 != 0, quads = p.quads && !spread;
    const int share = (k_blocks + WAVES - 1) / WAVES, begin = spread ? wave : wave * share, end = spread ? k_blocks : min(begin + share, k_blocks), stride = spread ? WAVES : 1;
    auto ask = [&](int i, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NT * 2; ++t) load_to_lds(rw, w_off[t], (unsigned) kb * 128u, lds0 + t * 1024);
#pragma unroll
        for (int t = 0; t < AM / 8; ++t) load_to_lds(ra, a_off[t], (unsigned) kb * 128u, lds0 + NT * 2048 + t * 1024);
        const unsigned to = lds0 + NT * 2048 + AM * 128 + (i / 4 & 1) * CHUNK;
        if (!quads) word_to_lds(scales + kb * scale_step, to + i % 4 * 256);
        else if (i % 4 == 0) quad_to_lds(scales + min(kb, k_blocks - 4), to);   // of four blocks, the last four as they are
    };
    const int row_step = quads ? 16 : 4;
    f32x4 acc[NT][MT] = {};
    if (begin < end) ask(0, begin);
    const char *slot = lds + wave * SLOT;
    for (int i = 0, kb = begin; kb < end; ++i, kb += stride) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        i32x4 w[NT][2], a[MT][2];
        float s[MT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int u = 0; u < NT; ++u) w[u][h] = *reinterpret_cast<const i32x4 *>(slot + (u * 16 + li) * 128 + (lane_unit(lq, h) ^ (li / 2)) * 16);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int row = AM < 16 ? li % AM : t * 16 + li;   // columns past the last row are not stored
                a[t][h] = *reinterpret_cast<const i32x4 *>(slot + NT * 2048 + row * 128 + (lane_unit(lq, h) ^ (row / 2 % 8)) * 16);
            }
        }
        const int first = kb - i % 4;
        const char *factor = slot + NT * 2048 + AM * 128 + (i / 4 & 1) * CHUNK + (quads ? (kb - min(first, k_blocks - 4)) * 4 : i % 4 * 256);
        const float sw = *reinterpret_cast<const float *>(factor + AM * row_step);
#pragma unroll
        for (int t = 0; t < MT; ++t) s[t] = *reinterpret_cast<const float *>(factor + (AM < 16 ? li % AM : t * 16 + li) * row_step) * sw;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read, so that the place can take another block
        if (kb + stride < end) ask(i + 1, kb + stride);
        if (kb * 128 + 128 > p.k) {   // the last block: nothing behind a row's end takes part
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int keep = p.k - (kb * 128 + lane_unit(lq, h) * 16);
#pragma unroll
                for (int u = 0; u < NT; ++u) w[u][h] = f8_kept(w[u][h], keep);
#pragma unroll
                for (int t = 0; t < MT; ++t) a[t][h] = f8_kept(a[t][h], keep);
            }
        }
        f32x4 part[NT][MT] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                bf16x8 y[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) y[t] = f8_widened(a[t][h][2 * e], a[t][h][2 * e + 1]);
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    const bf16x8 x = f8_widened(w[u][h][2 * e], w[u][h][2 * e + 1]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) part[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y[t], part[u][t], 0, 0, 0);
                }
            }
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[u][t][i] = __builtin_fmaf(part[u][t][i], s[t], acc[u][t][i]);
    }
    __syncthreads();
    f32x4 *parts = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t) parts[((wave * NT + u) * MT + t) * 64 + lane] = acc[u][t];
    __syncthreads();
    // a wavefront has tiles wave, wave + 8, ...: four consecutive outputs of a row a lane
#pragma unroll
    for (int i = 0; i < (NT * MT + WAVES - 1) / WAVES; ++i) {
        const int tile = wave + WAVES * i, u = tile / MT, t = tile % MT;
        if (tile >= NT * MT) break;
        f32x4 v = parts[tile * 64 + lane];
#pragma unroll
        for (int x = 1; x < WAVES; ++x) v += parts[(x * NT * MT + tile) * 64 + lane];
        const int m = t * 16 + li, n = n0 + u * 16 + lq * 4;
        if (m < rows_m && n < p.n) store4<DT>(p, m0 + m, n, v);
    }
#endif
}

// ---- many rows -----------------------------------------------------------------------------------------------------
// A workgroup a compute unit walks over tiles of 256 weights x 256 rows, eight wavefronts of 128 x 64: 2048 cycles of matrix instructions a block of channels, whose tiles come in during the
// block before, across the ends of tiles.  A matrix instruction has four multiply-adds beside it, which a SIMD with two wavefronts issues in its time but for a seventh (37 cycles for 32).
// 8192 rows of 4096 channels, 22016 outputs: 681 to 690 us, 2.15 PFLOP/s; 8192 of 8192, 8192 outputs 452 us, 2.43 PFLOP/s.  (Instructions alone reach 4.3 to 4.9 in a loop; the clock falls to some 2 GHz.)
// Measured and not kept: a block's last products held back over the barrier, loads a block and a half ahead with two barriers a block (8192^3 486 us), lines asked for ahead of time, stores past the
// caches (650 us with operands in the last-level cache, 701 with operands from memory).
__device__ __forceinline__ f32x4 f8_mma(i32x8 a, i32x8 b) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{}, 0, 0, 0, 0, 0, 0);
#else
    return {};
#endif
}

constexpr int HIGH = 6;   // rows of tiles that go together: 32 workgroups of an XCD share 6 + 6 panels at a time (2 or 8 some percent slower, 16 and 32 much)

template <int DT>
__global__ __launch_bounds__(512) void f8_many_kernel(const F8LinearParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BN = 256, BM = 256, WM = 4, TN = 8, TM = 4, TILES = (BN + BM) * 128, CHUNK = (BM + 64) * 16, STORES = TN * TM / 2;
    __shared__ __attribute__((aligned(1024))) char lds[2 * TILES + 2 * CHUNK];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lq = lane >> 4, wn = wave / WM, wm = wave % WM;
    const unsigned lds0 = (unsigned) (size_t) (__attribute__((address_space(3))) char *) lds;
    const int k_blocks = (p.k + 127) / 128, k16 = (p.k + 15) & ~15, blocks_n = (p.n + 127) / 128;
    // an XCD has a run of the tiles, HIGH rows of tiles by columns; its workgroups take them in turn
    const int tiles = p.tiles_m * p.tiles_n, xcd = (int) blockIdx.x & 7, each = tiles >> 3, over = tiles & 7;
    const int begin = xcd * each + min(xcd, over), end = begin + each + (xcd < over), step = ((int) gridDim.x - xcd + 7) >> 3;

    // what is loaded next: block `kb` of tile `lid`
    struct {
        int lid, kb, n0, m0, chunk;
        i32x4 w, a;
    } next;
    // a load's eight rows are row 32 wave + 8 i on, whose units are exchanged one way for even i and another for odd; rows behind a tile's last are behind its memory's end
    const int lrow = lane / 8, even = (lane % 8) ^ (lrow / 2), srow = wave * 64 + lane;
    const unsigned w_off[2] = {(unsigned) ((wave * 32 + lrow) * p.ws) + even * 16, (unsigned) ((wave * 32 + lrow) * p.ws) + (even ^ 4) * 16};
    const unsigned a_off[2] = {(unsigned) ((wave * 32 + lrow) * p.as) + even * 16, (unsigned) ((wave * 32 + lrow) * p.as) + (even ^ 4) * 16};
    const float *scales;
    const bool of_rows = wave < BM / 64;
    const long long scale_step = of_rows ? p.a_ss[1] : p.w_ss[1];
    auto set_tile = [&](int lid) __attribute__((always_inline)) {
        const bool live = lid < end;   // behind the last one nothing is fetched
        const int at = live ? lid : begin, group = (int) div31((unsigned) at, p.by_group), left = at - group * HIGH * p.tiles_n;
        const bool whole = group * HIGH + HIGH <= p.tiles_m;
        const int high = whole ? HIGH : p.tiles_m - group * HIGH, tn = whole ? left / HIGH : (int) div31((unsigned) left, p.by_last);
        next.lid = lid;
        next.kb = 0;
        next.n0 = tn * BN;
        next.m0 = (group * HIGH + left - tn * high) * BM;
        const int rows_n = min(BN, p.n - next.n0), rows_m = min(BM, p.m - next.m0);
        next.w = descriptor(p.w + (long long) next.n0 * p.ws, live ? (unsigned) ((rows_n - 1) * p.ws + k16) : 0u);
        next.a = descriptor(p.a + (long long) next.m0 * p.as, live ? (unsigned) ((rows_m - 1) * p.as + k16) : 0u);
        scales = of_rows ? p.a_scale + (next.m0 + min(srow, rows_m - 1)) * p.a_ss[0] : p.w_scale + min(next.n0 / 128 + lane, blocks_n - 1) * p.w_ss[0];
    };
    auto load_tiles = [&](int i, int buf) __attribute__((always_inline)) {   // an eighth of the block, i = 0 .. 7
        unsigned down = (unsigned) (i < 4 ? i * 8 * p.ws : (i - 4) * 8 * p.as);
        asm volatile("" : "+s"(down));   // added here, not kept in a register for each i
        if (i < 4) load_to_lds(next.w, w_off[i % 2] + down, (unsigned) next.kb * 128u, lds0 + buf * TILES + (wave * 4 + i) * 1024);
        else load_to_lds(next.a, a_off[i % 2] + down, (unsigned) next.kb * 128u, lds0 + buf * TILES + BN * 128 + (wave * 4 + i - 4) * 1024);
    };
    // scales, of four blocks at a time where they lie side by side (the last four of a row as they are)
    auto load_scales = [&]() __attribute__((always_inline)) {
        if (wave > BM / 64) return;
        const unsigned to = lds0 + 2 * TILES + next.chunk * CHUNK;
        if (p.quads) {
            if (next.kb % 4 == 0) quad_to_lds(scales + min(next.kb, k_blocks - 4), to + wave * 1024);
        } else {
            word_to_lds(scales + next.kb * scale_step, to + next.kb % 4 * ((BM + 64) * 4) + wave * 256);
        }
    };
    auto advance = [&]() __attribute__((always_inline)) {
        if (++next.kb == k_blocks) set_tile(next.lid + step);
        next.chunk ^= (int) ((unsigned) ((next.kb & 3) - 1) >> 31);   // every fourth block
    };

    next.chunk = 0;
    set_tile(begin + ((int) blockIdx.x >> 3));
    load_scales();
#pragma unroll
    for (int i = 0; i < 8; ++i) load_tiles(i, 0);
    int buf = 0, chunk = 1;
    bool stored = false;
    while (next.lid < end) {
        const int n0 = next.n0, m0 = next.m0;
        f32x4 acc[TN][TM] = {};
        for (int kb = 0; kb < k_blocks; ++kb, buf ^= 1) {
            // this block is there, and everybody has read the one before it; the last tile's results are on their way behind it
            if (stored) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(STORES) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            stored = false;
            char *stage = lds + buf * TILES;
            const int there = p.k - kb * 128;
            if (there < 128) {   // the last block: nothing behind a row's end takes part
                for (int i = threadIdx.x; i < (BN + BM) * 8; i += 512) {
                    const int row = i / 8, keep = there - ((i % 8) ^ (row / 2 % 8)) * 16;
                    if (keep >= 16) continue;
                    i32x4 *at = reinterpret_cast<i32x4 *>(stage + i * 16);
                    *at = f8_kept(*at, keep);
                }
                __syncthreads();
            }
            chunk ^= (int) ((unsigned) ((kb & 3) - 1) >> 31);
            const int first = p.quads ? min(kb & ~3, k_blocks - 4) : kb & ~3;   // of the chunk
            const char *factors = lds + 2 * TILES + chunk * CHUNK + (kb - first) * (p.quads ? 4 : (BM + 64) * 4);
            const int row_step = p.quads ? 16 : 4;
            auto operand = [&](int row) __attribute__((always_inline)) {
                const int swz = row / 2 % 8;
                const i32x4 x = *reinterpret_cast<const i32x4 *>(stage + row * 128 + (lane_unit(lq, 0) ^ swz) * 16), y = *reinterpret_cast<const i32x4 *>(stage + row * 128 + (lane_unit(lq, 1) ^ swz) * 16);
                return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            };
            // multiply-adds of a tile three matrix instructions behind it: its result is there, and the vector pipe works next to the matrix cores
            constexpr int BACK = 3;
            i32x8 a[3], b[TM];
            f32x4 part[BACK + 1];
            float s[TM];
            auto add = [&](int j) __attribute__((always_inline)) {
                const int u = j / TM, t = j % TM;
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[u][t][r] = __builtin_fmaf(part[j % (BACK + 1)][r], s[t], acc[u][t][r]);
            };
            advance();
            load_scales();
            __builtin_amdgcn_sched_barrier(0);
            a[0] = operand(wn * 128 + li);
#pragma unroll
            for (int t = 0; t < TM; ++t) b[t] = operand(BN + wm * 64 + t * 16 + li);
            __builtin_amdgcn_sched_barrier(0);
            const float sw = *reinterpret_cast<const float *>(factors + (BM + wn) * row_step);
#pragma unroll
            for (int t = 0; t < TM; ++t) s[t] = *reinterpret_cast<const float *>(factors + (wm * 64 + t * 16 + li) * row_step);
            a[1] = operand(wn * 128 + 16 + li);
#pragma unroll
            for (int u = 0; u < TN; ++u) {   // one basic block: across branches the multiply-adds would be put off
                if (u + 2 < TN) a[(u + 2) % 3] = operand(wn * 128 + (u + 2) * 16 + li);
#pragma unroll
                for (int t = 0; t < TM; ++t) {
                    const int j = u * TM + t;
                    __builtin_amdgcn_sched_barrier(0);
                    part[j % (BACK + 1)] = f8_mma(a[u % 3], b[t]);
                    if (j < TM) s[j] *= sw;
                    if (j >= BACK) add(j - BACK);
                    if (j < 16 && j % 2 == 1) load_tiles(j / 2, buf ^ 1);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = TN * TM - BACK; j < TN * TM; ++j) add(j);
        }

        // a lane has outputs 4 lq .. 4 lq + 3 of each tile, of row li
        int l = lane;
        asm volatile("" : "+v"(l));   // places in the result are worked out here, not kept over the blocks
        const int row = wm * 64 + (l & 15), n_lane = n0 + wn * 128 + (l >> 4) * 4;
        const int rows = min(BM, p.m - m0);
        const rsrc_t ro = make_rsrc(p.out + m0 * p.os, (unsigned) ((rows - 1) * p.os + p.n * 2));
        if (p.bias)
#pragma unroll
            for (int u = 0; u < TN; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float bias = n_lane + u * 16 + i < p.n ? p.bias[n_lane + u * 16 + i] : 0.0f;
#pragma unroll
                    for (int t = 0; t < TM; ++t) acc[u][t][i] += bias;
                }
        // two tiles' halves exchanged between groups of lanes: eight consecutive outputs a lane
        const int n_wide = n0 + wn * 128 + (l >> 4) % 2 * 16 + (l >> 5) * 8;
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const bool live = row + t * 16 < rows;
            const unsigned off = (unsigned) ((row + t * 16) * p.os) + n_wide * 2;
#pragma unroll
            for (int u = 0; u < TN; u += 2) {
                unsigned x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[i] = pack_h16<DT>(acc[u][t][2 * i], acc[u][t][2 * i + 1]);
                    y[i] = pack_h16<DT>(acc[u + 1][t][2 * i], acc[u + 1][t][2 * i + 1]);
                    const auto z = __builtin_amdgcn_permlane16_swap(x[i], y[i], false, false);
                    x[i] = z[0];
                    y[i] = z[1];
                }
                const bool there = live && n_wide + u * 16 + 8 <= p.n;
                if (p.wide) __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], x[1], y[0], y[1]}, ro, there ? off + u * 32 : OOB, 0, 0);
                else if (there) *reinterpret_cast<any_u32x4 *>(p.out + m0 * p.os + off + u * 32) = any_u32x4{x[0], x[1], y[0], y[1]};
            }
        }
        stored = p.wide;
        const int from = p.n & ~7;   // the last ones of a row, one at a time
        if (from < p.n && n0 + BN > from) {
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                const unsigned off = row + t * 16 < rows ? (unsigned) ((row + t * 16) * p.os) : OOB;
#pragma unroll
                for (int u = 0; u < TN; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int n = n_lane + u * 16 + i;
                        __builtin_amdgcn_raw_buffer_store_b16((unsigned short) pack_h16<DT>(acc[u][t][i], 0.0f), ro, n >= from && n < p.n ? off + n * 2 : OOB, 0, 0);
                    }
            }
            stored = false;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // loads that wrote nothing but zeros are still on their way to LDS
#endif
}

// ---- some rows -----------------------------------------------------------------------------------------------------
// A workgroup has BN weights x BM rows, its wavefronts WN x WM parts of them in each of KG groups, and a group a run of the blocks of channels, in a ring of DEPTH blocks: tiles
// enough for the compute units, and wavefronts enough for a unit, where there are few rows.  The groups' sums meet in LDS, in one order.
// EXACT: matrix instructions in bf16, which sum in fp32: for fp32 results, and for 16-bit ones where they are asked for.
// Bound by what goes into LDS: a block of 96 x 64 is 20 KB for 192 cycles of matrix instructions, and takes some 800.  300 rows of 11008 channels, 4096 outputs 38 us with weights from memory (0.7 PFLOP/s,
// 215 tiles on 256 units), 26 to 30 from the last-level cache.  Measured and not kept: operands of the next block read ahead into registers, lines asked for ahead of time (2 to 15% behind).
template <int DT, bool EXACT, int BN, int BM, int KG, int WN, int WM, int DEPTH>
__global__ __launch_bounds__(64 * KG * WN * WM) void f8_tile_kernel(const F8LinearParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int GW = WN * WM, TN = BN / WN / 16, TM = BM / WM / 16, LN = BN / 8 / GW, LM = BM / 8 / GW, LOADS = LN + LM;
    constexpr int SLOT = (BN + BM) * 128, CHUNK = (BM + 64) * 16, RING = KG * (DEPTH * SLOT + 2 * CHUNK), JOIN = KG * GW * TN * TM * 1024;
    constexpr bool ONE = 128 % (BN / WN) == 0;   // a wavefront's weights share a scale; else sixteen of them do
    static_assert(BN % (16 * WN) == 0 && BM % 64 == 0 && BM / 64 < GW && LN >= 1 && LM >= 1, "64 rows' scales are a wavefront's load, those of the weights another's, and every wavefront loads");
    __shared__ __attribute__((aligned(1024))) char lds[RING > JOIN ? RING : JOIN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lq = lane >> 4, kg = wave / GW, gw = wave % GW, wn = gw / WM, wm = gw % WM;
    int n0, m0;
    {   // an XCD has a run of the tiles, all rows of a column of them by the next
        const int bid = blockIdx.x, nb = (int) gridDim.x, q = nb >> 3, rem = nb & 7, xcd = bid & 7;
        const unsigned lid = (unsigned) (xcd * q + min(xcd, rem) + (bid >> 3)), tn = div31(lid, p.by_last);
        n0 = (int) tn * BN;
        m0 = (int) (lid - tn * (unsigned) p.tiles_m) * BM;
    }
    const int k_blocks = (p.k + 127) / 128, k16 = (p.k + 15) & ~15, rows_n = min(BN, p.n - n0), rows_m = min(BM, p.m - m0);
    const char *w_base = p.w + (long long) n0 * p.ws, *a_base = p.a + (long long) m0 * p.as;
    const unsigned w_bytes = (unsigned) ((rows_n - 1) * p.ws + k16), a_bytes = (unsigned) ((rows_m - 1) * p.as + k16);
    unsigned w_off[LN], a_off[LM];
    const int lrow = lane / 8;
#pragma unroll
    for (int t = 0; t < LN; ++t) {
        const int row = (gw * LN + t) * 8 + lrow;
        w_off[t] = row < rows_n ? (unsigned) (row * p.ws) + ((lane % 8) ^ (row / 2 % 8)) * 16 : OOB;
    }
#pragma unroll
    for (int t = 0; t < LM; ++t) {
        const int row = (gw * LM + t) * 8 + lrow;
        a_off[t] = row < rows_m ? (unsigned) (row * p.as) + ((lane % 8) ^ (row / 2 % 8)) * 16 : OOB;
    }
    // a lane's scale: of 64 rows a wavefront, of the weights' blocks of 128 in the one behind those
    constexpr int OWN = BM / WM;
    const int n_wave = n0 + wn * (BN / WN), m_wave = m0 + wm * OWN, blocks_n = (p.n + 127) / 128;
    const bool of_rows = gw < BM / 64;
    const float *scales = of_rows ? p.a_scale + (m0 + min(gw * 64 + lane, rows_m - 1)) * p.a_ss[0] : p.w_scale + min(n0 / 128 + lane, blocks_n - 1) * p.w_ss[0];
    const long long scale_step = of_rows ? p.a_ss[1] : p.w_ss[1];
    const unsigned lds0 = (unsigned) (size_t) (__attribute__((address_space(3))) char *) lds + kg * DEPTH * SLOT;
    const unsigned scales0 = (unsigned) (size_t) (__attribute__((address_space(3))) char *) lds + KG * DEPTH * SLOT + kg * 2 * CHUNK;
    const int share = (k_blocks + KG - 1) / KG, begin = kg * share, end = min(begin + share, k_blocks);
    auto ask_scales = [&](int i) __attribute__((always_inline)) {   // in front of the block's others: a wait for those is one for it
        const int kb = begin + i;
        if (kb >= end || gw > BM / 64) return;
        const unsigned chunk = scales0 + (i / 4 & 1) * CHUNK;
        if (!p.quads) word_to_lds(scales + kb * scale_step, chunk + i % 4 * (CHUNK / 4) + gw * 256);
        else if (i % 4 == 0) quad_to_lds(scales + min(kb, k_blocks - 4), chunk + gw * 1024);
    };
    auto ask = [&](int j, int i, int d) __attribute__((always_inline)) {   // j = 0 .. LOADS - 1
        const bool live = begin + i < end;   // one that is not there is not fetched
        const unsigned from = live ? (unsigned) (begin + i) * 128u : 0u, to = lds0 + d * SLOT;
        if (j < LN) load_to_lds(descriptor(w_base, live ? w_bytes : 0u), w_off[j], from, to + (gw * LN + j) * 1024);
        else load_to_lds(descriptor(a_base, live ? a_bytes : 0u), a_off[j - LN], from, to + BN * 128 + (gw * LM + j - LN) * 1024);
    };
    const int row_step = p.quads ? 16 : 4;
    f32x4 acc[TN][TM] = {};
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) {
        ask_scales(d);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) ask(j, d, d);
    }
    for (int first = 0; first < share; first += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int i = first + d, kb = begin + i;
            if (i >= share) break;   // uniform over the workgroup
            // this block is there, and everybody has read the one before it
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((DEPTH - 2) * LOADS) : "memory");
            const int then = i + DEPTH - 1;
            ask_scales(then);
            if (kb >= end) {
#pragma unroll
                for (int j = 0; j < LOADS; ++j) ask(j, then, (d + DEPTH - 1) % DEPTH);
                continue;
            }
            const char *slot = lds + (kg * DEPTH + d) * SLOT;
            const char *factor = lds + KG * DEPTH * SLOT + (kg * 2 + (i / 4 & 1)) * CHUNK + (p.quads ? (kb - min(kb - i % 4, k_blocks - 4)) * 4 : i % 4 * (CHUNK / 4));
            float s[TM], sw[TN];
#pragma unroll
            for (int u = 0; u < (ONE ? 1 : TN); ++u) sw[u] = *reinterpret_cast<const float *>(factor + (BM + (n_wave + u * 16) / 128 - n0 / 128) * row_step);
#pragma unroll
            for (int t = 0; t < TM; ++t) s[t] = *reinterpret_cast<const float *>(factor + (wm * OWN + t * 16 + li) * row_step) * (ONE ? sw[0] : 1.0f);
            i32x4 a[TN][2], b[TM][2];
            auto operand = [&](int row, i32x4 (&x)[2]) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) x[h] = *reinterpret_cast<const i32x4 *>(slot + row * 128 + (lane_unit(lq, h) ^ (row / 2 % 8)) * 16);
            };
#pragma unroll
            for (int t = 0; t < TM; ++t) operand(BN + wm * OWN + t * 16 + li, b[t]);
#pragma unroll
            for (int u = 0; u < TN; ++u) operand(wn * (BN / WN) + u * 16 + li, a[u]);
            if (kb * 128 + 128 > p.k) {   // the last block: nothing behind a row's end takes part
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int keep = p.k - (kb * 128 + lane_unit(lq, h) * 16);
#pragma unroll
                    for (int u = 0; u < TN; ++u) a[u][h] = f8_kept(a[u][h], keep);
#pragma unroll
                    for (int t = 0; t < TM; ++t) b[t][h] = f8_kept(b[t][h], keep);
                }
            }
            // loads between the matrix instructions: a wavefront stands still where it asks for more than the memory pipe takes at once
            f32x4 part[TN][TM] = {};
            auto step = [&](int j) __attribute__((always_inline)) {
                __builtin_amdgcn_sched_barrier(0);
                if (j < LOADS) ask(j, then, (d + DEPTH - 1) % DEPTH);
            };
            static_assert(LOADS <= TN * TM, "a load behind each product");
            if constexpr (EXACT) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        bf16x8 y[TM];
#pragma unroll
                        for (int t = 0; t < TM; ++t) y[t] = f8_widened(b[t][h][2 * e], b[t][h][2 * e + 1]);
#pragma unroll
                        for (int u = 0; u < TN; ++u) {
                            const bf16x8 x = f8_widened(a[u][h][2 * e], a[u][h][2 * e + 1]);
#pragma unroll
                            for (int t = 0; t < TM; ++t) {
                                part[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y[t], part[u][t], 0, 0, 0);
                                if (h == 0 && e == 0) step(u * TM + t);
                            }
                        }
                    }
            } else {
#pragma unroll
                for (int u = 0; u < TN; ++u)
#pragma unroll
                    for (int t = 0; t < TM; ++t) {
                        part[u][t] = f8_mma(__builtin_shufflevector(a[u][0], a[u][1], 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(b[t][0], b[t][1], 0, 1, 2, 3, 4, 5, 6, 7));
                        step(u * TM + t);
                    }
            }
#pragma unroll
            for (int u = 0; u < TN; ++u)
#pragma unroll
                for (int t = 0; t < TM; ++t) {
                    const float by = ONE ? s[t] : s[t] * sw[u];
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[u][t][i] = __builtin_fmaf(part[u][t][i], by, acc[u][t][i]);
                }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // loads that wrote nothing but zeros are still on their way to LDS
    __syncthreads();
    f32x4 *parts = reinterpret_cast<f32x4 *>(lds);
    if constexpr (KG > 1) {
#pragma unroll
        for (int u = 0; u < TN; ++u)
#pragma unroll
            for (int t = 0; t < TM; ++t) parts[(wave * TN * TM + u * TM + t) * 64 + lane] = acc[u][t];
        __syncthreads();
    }
    // a lane has four consecutive outputs of a row; the groups share the tiles out
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const int j = u * TM + t;
            if (KG > 1 && j % KG != kg) continue;   // uniform
            f32x4 v = acc[u][t];
            if constexpr (KG > 1) {
                v = parts[(gw * TN * TM + j) * 64 + lane];
#pragma unroll
                for (int g = 1; g < KG; ++g) v += parts[((g * GW + gw) * TN * TM + j) * 64 + lane];
            }
            const int m = m_wave + t * 16 + li, n = n_wave + u * 16 + lq * 4;
            if (m < p.m && n < p.n) store4<DT>(p, m, n, v);
        }
#endif
}

template <int DT, int AM, int NT, int WAVES> static int few_launch(const F8LinearParams &p, hipStream_t stream) {
    hipLaunchKernelGGL((f8_few_kernel<DT, AM, NT, WAVES>), dim3((unsigned) ((p.n + 16 * NT - 1) / (16 * NT)), (unsigned) ((p.m + AM - 1) / AM)), dim3(64 * WAVES), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

template <int DT> static int many_launch(F8LinearParams p, hipStream_t stream) {
    p.tiles_n = (p.n + 255) / 256;
    p.tiles_m = (p.m + 255) / 256;
    const long long tiles = (long long) p.tiles_n * p.tiles_m;
    if (tiles >= 1LL << 31) return set_error(ONHIP_ERR_ARG, "e4m3 product: %lld tiles", tiles);
    p.by_group = make_div31((unsigned) (HIGH * p.tiles_n));
    p.by_last = make_div31((unsigned) (p.tiles_m % HIGH ? p.tiles_m % HIGH : HIGH));
    hipLaunchKernelGGL((f8_many_kernel<DT>), dim3((unsigned) (tiles < 256 ? tiles : 256)), dim3(512), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

template <int DT, bool EXACT, int BN, int BM, int KG, int WN, int WM, int DEPTH> static int tile_launch(F8LinearParams p, hipStream_t stream) {
    p.tiles_n = (p.n + BN - 1) / BN;
    p.tiles_m = (p.m + BM - 1) / BM;
    p.by_last = make_div31((unsigned) p.tiles_m);
    const long long tiles = (long long) p.tiles_n * p.tiles_m;
    constexpr int THREADS = 64 * KG * WN * WM;
    if (tiles * THREADS >= 1LL << 32) return set_error(ONHIP_ERR_ARG, "e4m3 product: %lld tiles", tiles);   // a launch's threads
    hipLaunchKernelGGL((f8_tile_kernel<DT, EXACT, BN, BM, KG, WN, WM, DEPTH>), dim3((unsigned) tiles), dim3(THREADS), 0, stream, p);
    ONHIP_CHECK_HIP(hipGetLastError());
    return ONHIP_OK;
}

// What a product of more than 32 rows runs on: the least expected time, as rounds of tiles over the 256 compute units (PAIR: two workgroups a unit) times what a block of channels was
// measured to take there, in us, with weights that come from memory, at 4096 outputs of 4096 channels and 33 to 2048 rows (mostly within a tenth for 22016 outputs and 11008 channels).
// Sums of 13 bits, bf16 results: 256 rows of 4096 channels, 4096 outputs 22, 14, 16, 18, 19, 28, 38 and 62 us in this order; 400 rows, 6144 outputs 43, 36, 29, 32, 26, 28, 38 and 60; 1024 rows, 4096 outputs 63,
// 50, 44, 36, 40, 29, 38 and 61; 2048 rows 117, 104, 87, 72, 69, 55, 46 and 62; 300 rows of 11008 channels 56, 56, 38, 44, 44, 64, 89 and 143; 512 rows of 4096, 22016 outputs 198, 136, 116,
// 106, 95, 82, 83 and 65.  Exact sums, fp32 results: 700 rows of 11008, 4096 outputs 117, 104, 90, 106, 83 and, in pairs, 101
enum { BY_FEW, BY_64, BY_96, BY_128, BY_96_PAIR, BY_SQUARE, BY_SQUARE_PAIR, BY_MANY };
static int linear_choice(const F8LinearParams &p, bool exact) {
    constexpr float never = 1e9f;                                     // 128 x 128 in bf16 takes alone what it takes in pairs, up to 256 of them
    static constexpr struct {
        int n, m, slots;
        float one, full, exact_one, exact_full, round;   // a block: of a round of up to 256 workgroups, of a full one; in bf16; once a round
    } ways[] = {{32, 32, 512, 0.15f, 0.26f, 0.15f, 0.27f, 1.0f}, {64, 64, 256, 0.32f, 0.32f, 0.40f, 0.40f, 1.0f}, {96, 64, 256, 0.38f, 0.38f, 0.53f, 0.53f, 1.0f},
                {128, 64, 256, 0.46f, 0.46f, 0.62f, 0.62f, 1.0f}, {96, 64, 512, 0.44f, 0.67f, 0.62f, 0.93f, 1.5f}, {128, 128, 256, 0.73f, 0.73f, never, never, 1.5f}, {128, 128, 512, 1.00f, 1.30f, 1.12f, 1.95f, 1.5f},
                {256, 256, 256, 1.65f, 1.65f, never, never, 6.0f}};
    const float blocks = (float) ((p.k + 127) / 128);
    int best = BY_SQUARE_PAIR;
    float least = INFINITY;
    for (int i = 0; i <= BY_MANY; ++i) {
        if (exact && ways[i].exact_one == never) continue;
        if (i == BY_MANY && p.os > (1 << 22)) break;               // a tile's results within 2^30 bytes
        if (i == BY_FEW && p.m > 32 * 65535) continue;             // groups of rows are the grid's second dimension
        const long long tiles = ((long long) (p.n + ways[i].n - 1) / ways[i].n) * ((p.m + ways[i].m - 1) / ways[i].m), rounds = tiles / ways[i].slots, rest = tiles % ways[i].slots;
        const float one = exact ? ways[i].exact_one : ways[i].one, full = exact ? ways[i].exact_full : ways[i].full;
        const float t = (float) rounds * (full * blocks + ways[i].round) + (rest == 0 ? 0.0f : (rest <= 256 ? one : full) * blocks + ways[i].round);
        if (t < least) {
            best = i;
            least = t;
        }
    }
    return best;
}

static int linear_check(const onhip_f8_linear_desc_t *d, int *dt) {
    const char *what = "e4m3 product";
    constexpr int MOST = 1 << 27;
    if (!d || d->rows < 1 || d->outputs < 1 || d->channels < 1) return set_error(ONHIP_ERR_ARG, "%s: bad shape", what);
    if (!element_type(d->compute, dt)) return set_error(ONHIP_ERR_ARG, "%s: unknown type %d", what, d->compute);
    if (d->exact != 0 && d->exact != 1) return set_error(ONHIP_ERR_ARG, "%s: exact = %d", what, d->exact);
    if (d->rows > MOST || d->outputs > MOST || d->channels > (1 << 22)) return set_error(ONHIP_ERR_ARG, "%s: %d rows, %d outputs, %d channels (up to 2^27, 2^27, 2^22)", what, d->rows, d->outputs, d->channels);
    // byte offsets within a tile stay below 2^31
    const long long most = 1LL << 22;
    if (d->rows > 1 && (d->a_stride < d->channels || d->a_stride > most || d->a_stride % 16)) return set_error(ONHIP_ERR_ARG, "%s: rows %lld bytes apart (a multiple of 16, up to 2^22)", what, d->a_stride);
    if (d->outputs > 1 && (d->w_stride < d->channels || d->w_stride > most || d->w_stride % 16)) return set_error(ONHIP_ERR_ARG, "%s: weights %lld bytes apart (a multiple of 16, up to 2^22)", what, d->w_stride);
    if (d->rows > 1 && (d->out_stride < d->outputs || d->out_stride > (1LL << 40))) return set_error(ONHIP_ERR_ARG, "%s: results %lld elements apart", what, d->out_stride);
    const int blocks = (d->channels + F8_BLOCK - 1) / F8_BLOCK, blocks_n = (d->outputs + F8_BLOCK - 1) / F8_BLOCK, extent[4] = {d->rows, blocks, blocks_n, blocks};
    for (int i = 0; i < 4; ++i) {
        const long long stride = i < 2 ? d->a_scale_strides[i] : d->w_scale_strides[i - 2];
        if (extent[i] > 1 && (stride < 0 || stride > (1LL << 40))) return set_error(ONHIP_ERR_ARG, "%s: bad scale strides", what);
    }
    return ONHIP_OK;
}

// sizes and strides; 0 for a stride that is never stepped over
static F8LinearParams linear_shape(const onhip_f8_linear_desc_t *d, int size) {
    F8LinearParams p = {};
    p.m = d->rows;
    p.n = d->outputs;
    p.k = d->channels;
    p.as = d->rows > 1 ? (int) d->a_stride : 0;
    p.ws = d->outputs > 1 ? (int) d->w_stride : 0;
    p.os = d->rows > 1 ? d->out_stride * size : 0;
    const int blocks = (p.k + F8_BLOCK - 1) / F8_BLOCK;
    p.a_ss[0] = p.m > 1 ? d->a_scale_strides[0] : 0;
    p.a_ss[1] = blocks > 1 ? d->a_scale_strides[1] : 0;
    p.w_ss[0] = p.n > F8_BLOCK ? d->w_scale_strides[0] : 0;
    p.w_ss[1] = blocks > 1 ? d->w_scale_strides[1] : 0;
    p.quads = blocks >= 4 && p.a_ss[1] == 1 && p.w_ss[1] == 1;
    return p;
}

}  // namespace onhip

using namespace onhip;

extern "C" {

int onhip_linear_f8_way(const onhip_f8_linear_desc_t *d) {
    int dt;
    if (int rc = linear_check(d, &dt)) return rc;
    return d->rows <= 32 ? (int) BY_FEW : linear_choice(linear_shape(d, bytes_of(dt)), dt == DT_F32 || d->exact);
}

int onhip_linear_f8(const onhip_f8_linear_desc_t *d, const void *a, const float *a_scale, const void *w, const float *w_scale, const float *bias, void *out, void *stream) {
    const char *what = "e4m3 product";
    int dt;
    if (int rc = linear_check(d, &dt)) return rc;
    if (!a || !a_scale || !w || !w_scale || !out) return set_error(ONHIP_ERR_ARG, "%s: null pointer", what);
    if (misaligned(a, 16) || misaligned(w, 16)) return set_error(ONHIP_ERR_ARG, "%s: rows and weights must be 16-byte aligned", what);
    const int size = bytes_of(dt);
    if (misaligned(a_scale, 4) || misaligned(w_scale, 4) || misaligned(bias, 4) || misaligned(out, (uintptr_t) size)) return set_error(ONHIP_ERR_ARG, "%s: misaligned scales, bias or result", what);
    F8LinearParams p = linear_shape(d, size);
    const int blocks = (p.k + F8_BLOCK - 1) / F8_BLOCK, blocks_n = (p.n + F8_BLOCK - 1) / F8_BLOCK;
    const Span of_out = {static_cast<const char *>(out), p.os, (long long) p.n * size, p.m};
    for (const Span &from : {Span{static_cast<const char *>(a), p.as, p.k, p.m}, Span{static_cast<const char *>(w), p.ws, p.k, p.n}, scale_span(a_scale, p.a_ss, p.m, blocks), scale_span(w_scale, p.w_ss, blocks_n, blocks),
                             Span{reinterpret_cast<const char *>(bias), 0, 4LL * p.n, 1}})
        if (!apart(of_out, from)) return set_error(ONHIP_ERR_ARG, "%s: the result lies over an operand", what);
    p.a = static_cast<const char *>(a);
    p.w = static_cast<const char *>(w);
    p.a_scale = a_scale;
    p.w_scale = w_scale;
    p.bias = bias;
    p.out = static_cast<char *>(out);
    p.wide = !misaligned(out, 4) && p.os % 4 == 0;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    // up to 32 rows: 16 outputs a workgroup, or 32 and half as many wavefronts where that leaves four workgroups a compute unit (32003 outputs of 4000 channels, 5 rows: 28.8 and
    // 27.6 us; 4096 of 4096, 16 rows: 5.6 and 7.1; weights from the last-level cache.  Widths between those were not timed)
    auto few = [&]<int DT>() {
        const bool wide = p.n > 16384;
        if (p.m <= 8) return wide ? few_launch<DT, 8, 2, 4>(p, st) : few_launch<DT, 8, 1, 8>(p, st);
        if (p.m <= 16) return wide ? few_launch<DT, 16, 2, 4>(p, st) : few_launch<DT, 16, 1, 8>(p, st);
        if (p.m <= 32 && p.n <= 4096) return few_launch<DT, 32, 1, 8>(p, st);   // 32 rows of 11008 channels, 4096 outputs: 14.0 us, 17.2 with 32 outputs a workgroup
        return wide && p.m <= 32 ? few_launch<DT, 32, 2, 4>(p, st) : few_launch<DT, 32, 2, 8>(p, st);
    };
    auto by_sums = [&]<int DT, bool EXACT>() {
        if (p.m <= 32) return few.template operator()<DT>();
        switch (linear_choice(p, EXACT)) {
        case BY_FEW: return few.template operator()<DT>();
        case BY_64: return tile_launch<DT, EXACT, 64, 64, 2, 2, 2, 3>(p, st);
        case BY_96: return tile_launch<DT, EXACT, 96, 64, 2, 2, 2, 3>(p, st);
        case BY_128: return tile_launch<DT, EXACT, 128, 64, 2, 2, 2, 3>(p, st);
        case BY_96_PAIR: return tile_launch<DT, EXACT, 96, 64, 1, 2, 2, 3>(p, st);
        case BY_SQUARE_PAIR: return tile_launch<DT, EXACT, 128, 128, 1, 2, 2, 2>(p, st);
        case BY_SQUARE: if constexpr (!EXACT) return tile_launch<DT, EXACT, 128, 128, 1, 2, 2, 3>(p, st); break;
        case BY_MANY: if constexpr (!EXACT) return many_launch<DT>(p, st); break;
        }
        return set_error(ONHIP_ERR_ARG, "%s: no kernel", what);
    };
    auto go = [&]<int DT>() {
        if constexpr (DT != DT_F32)
            if (!d->exact) return by_sums.template operator()<DT, false>();
        return by_sums.template operator()<DT, true>();
    };
    return dt == DT_F32 ? go.template operator()<DT_F32>() : dt == DT_BF16 ? go.template operator()<DT_BF16>() : go.template operator()<DT_F16>();
}

}  // extern "C"
