// Attention of answers that share long prompts, over the 4-bit cache: a prompt's slots are read once for all of its
// answers.
//
// A row's softmax over its prompt's slots and its own is the join of parts: with a part's reference m_p, sum of weights
// l_p and sums o_p, out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p. A prompt's part has the rows of all its answers
// (answers x T x query heads of a kv head) in the MFMAs' N dimension, so a tile of slots is fetched and turned
// into bf16 once for 32 rows instead of once for each answer's 4 or 16; the answers' own slots are short lists, as in
// the attention of single lanes. Both kinds are blocks of one launch, and a second launch joins the parts. Where the lists are
// short, that costs more than it saves, and each answer's rows walk their prompt's tiles and their own in one launch.
//
// Times below of a kernel alone are a tracer's. Under it calls of two launches take up to 10 us longer than without (256 answers
// to 32,768 slots 91 for 81.5), so the two do not add up to the call's.
#include <algorithm>
#include <climits>

#include "q35_answers.h"
#include "q35_kv4_tile.h"

namespace q35 {

// A partial result of 16 rows, as the waves that end it hold it, so that stores and loads are whole runs (rows of dims in
// order, in pieces of 16 bytes from 64 lanes, took 5 us of 256 blocks' 17): row n's kRun dims from (4 g + r) D / 16 + w kRun on
// at kRun (64 (4 w + r) + 16 g + n), g, r, w < 4; then the rows' references and sums of weights.
template <int D>
constexpr int kRun = D / 64;
__host__ __device__ constexpr int tile_floats(int D) { return 16 * D + 32; }
long long kv4_shared_room(int D) { return (long long)(kv4_part_floats() / tile_floats(D)); }

// x / d for x d < 2^32, by d's reciprocal 2^32 / d + 1 (0 stands for d = 1): what the product has too much is under
// x / 2^32 < 1 / d. A launch's rows are at most 16 of the partial results' tiles, 129,072 of 64 dims, its T x group at most
// 32,768, its kv_heads and group 1024.
static uint32_t reciprocal(int d) { return d > 1 ? (uint32_t)(0x100000000ull / d + 1) : 0; }
__device__ __forceinline__ int over(int x, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)x, inv) : x; }

// Rows rho0 .. of the `rows` rows of the sorted sequences from `start` on, over tiles t0 .. t1 - 1 of a region.
struct Part {
    const uint8_t* region;
    int start, rows, rho0, h, t0, t1;
    int last;                        // the last slot of all rows, or -1: a row's own position, from pos on
    int pos;
    int tile;                        // where its rows go: tiles of partial results from here on
    const uint8_t* prefix;           // (both lists at once) the prompt's region, its slots and tiles: the list's first
    int len, ahead;
};

// A part: by a block's four waves, each every fourth tile, their states joined through LDS (W 4), or by a wave (1).
template <int D>
struct Exchange {                    // between a block's waves
    f32x4 os[4][4][D / 64][64];
    float ms[4][16], ls[4][16];
    uint32_t bs[4][16];
};
// BOTH: not a part, but all that the rows see, the prompt's tiles and then their own, and the end of it. The prompt's last
// tile comes first, as a few sinks before a window: the only one of the prompt's that may hold more than they see.
template <int D, int NQ, int W, bool BOTH = false>
__device__ __forceinline__ void part_rows(const Kv4Shared& a, const Part& p, uint32_t seqs, Exchange<D>& ex) {
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, nn = lane & 15, g = lane >> 4, group = a.q_heads / a.kv_heads;
    const float scale2 = fmaxf(fabsf(a.scale) * 1.44269504088896f, 0x1p-149f);      // (as in the attention of single lanes)
    const Lanes lo = lane_offsets<D>();
    const auto at = [&](int i) { return i; };
    const auto tile_at = [&](int i) {
        if (!BOTH) return p.region + (size_t)i * kv4_tile_bytes(D);
        return i < p.ahead ? p.prefix + (size_t)(i ? i - 1 : p.ahead - 1) * kv4_tile_bytes(D)
                           : p.region + (size_t)(i - p.ahead) * kv4_tile_bytes(D);
    };
    Tile<D> buf[kAhead<D>];
    first_tiles<D, NQ, W>(buf, p.t0, p.t1, tile_at, lo);
    const uint16_t* qrow[NQ];
    Sight sight[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int rho = min(p.rho0 + c * 16 + nn, p.rows - 1), i = over(rho, a.per_inv), r = rho - i * a.T * group;
        const int t = over(r, a.group_inv), s = p.start + i, seq = __shfl((int)seqs, s >> 2) >> 8 * (s & 3) & 255;
        qrow[c] = a.q.p + ((long long)seq * a.TT + t) * a.q.row + (p.h * group + r - t * group) * a.q.head;
        if (BOTH) sight[c] = {32 * p.ahead + p.pos + t, p.len & 31 ? 32 : 0, p.len & 31};
        else sight[c] = {p.last >= 0 ? p.last : p.pos + t, 0, 0};
    }
    const auto q_at = [&](int c, int gg, int k) {
        u32x4 w = *(const u32x4*)(qrow[c] + gg * (D / 4) + 8 * k);
        if (a.scale < 0.f) w ^= 0x80008000u;
        return __builtin_bit_cast(q35_bf16x8, w);
    };
    q35_bf16x8 qf[NQ == 1 ? D / 32 : 1];
    q35_bf16x8* ql = (q35_bf16x8*)&ex.os[0][0][0][0] + (W == 1 ? wv * NQ * (D / 32) * 64 : 0);
    if constexpr (NQ == 1) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k) qf[k] = q_at(0, g, k);
    } else {
#pragma unroll
        for (int c = 0; c < NQ; ++c)
#pragma unroll
            for (int k = 0; k < (D / 32 + W - 1) / W; ++k) {
                const int kk = W == 1 ? k : k * W + wv;
                if (kk < D / 32) ql[(c * (D / 32) + kk) * 64 + lane] = q_at(c, g, kk);
            }
        if (W > 1) lds_barrier();
        else wave_sync();
    }
    int qlane = lane;
    const auto q = [&](int c, int k) { return NQ == 1 ? qf[k] : ql[(c * (D / 32) + k) * 64 + qlane]; };
    const int full0 = BOTH && p.len & 31 ? 32 : 0;
    const int full1 = BOTH ? 32 * p.ahead + p.pos + over(p.rho0, a.group_inv) : p.last >= 0 ? p.last : p.pos + over(p.rho0, a.group_inv);
    Rows<D, NQ> st;
    walk_tiles<D, NQ, W>(st, buf, p.t0, p.t1, at, tile_at, lo, q, qlane, sight, full0, full1, scale2);
    if constexpr (BOTH) {
        join_waves<D, NQ, W>(st, p.rows - p.rho0, ex.os, ex.ms, ex.ls, ex.bs, [&](int c) {
            const int rho = min(p.rho0 + c * 16 + nn, p.rows - 1), t = over(rho, a.group_inv);
            const int seq = __builtin_amdgcn_readlane((int)seqs, p.start >> 2) >> 8 * (p.start & 3) & 255;
            const Out to(a, (long long)seq * a.TT + t, p.h * group + rho - t * group);
            return [=, &a](float (*x)[kRun<D>], float m, float sum) {
#pragma unroll
                for (int r = 0; r < 4; ++r) to.store<kRun<D>>(a, x[r], sum, first_dim<D, W>(r));
            };
        });
    } else if constexpr (W > 1) {
        join_waves<D, NQ, W>(st, p.rows - p.rho0, ex.os, ex.ms, ex.ls, ex.bs, [&](int c) {
            float* to = a.part + (size_t)(p.tile + c) * tile_floats(D);
            return [=](float (*x)[kRun<D>], float m, float sum) {
#pragma unroll
                for (int r = 0; r < 4; ++r) __builtin_memcpy(to + (64 * (4 * wv + r) + lane) * kRun<D>, x[r], 4 * kRun<D>);
                if (wv == 0 && g == 0) *(float2*)(to + 16 * D + 2 * nn) = make_float2(m, sum);
            };
        });
    } else {
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            uint32_t bad = st.bad[c];
            bad |= (uint32_t)__shfl_xor((int)bad, 16);
            bad |= (uint32_t)__shfl_xor((int)bad, 32);
            if (p.rho0 + c * 16 + nn >= p.rows) continue;
            float* to = a.part + (size_t)(p.tile + c) * tile_floats(D);
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x[kRun<D>];
#pragma unroll
                    for (int i = 0; i < kRun<D>; ++i)
                        x[i] = (bad >> ((4 * g + r) * (D / 16) + w * kRun<D>) / 32) & 1 ? __uint_as_float(0x7fc00000u) : st.o[c][w * kRun<D> + i][r];
                    __builtin_memcpy(to + (64 * (4 * w + r) + lane) * kRun<D>, x, 4 * kRun<D>);
                }
            if (g == 0) *(float2*)(to + 16 * D + 2 * nn) = make_float2(st.m[c], st.l[c][0]);
        }
    }
}

// The launch's entries and sequences as a wave holds them, an entry and four sequences a lane: the arrays are kernel
// arguments, cold in every cache at a launch, so all are fetched at once and picked from by lane. (Indexing them
// costs a trip to memory for each that depends on another, and was compiled wrongly: an int array's scalar load from an
// address that shares the index of a 16-bit one, whose low bit the hardware drops.)
struct Entries {
    int first, part, len, tile, lane, start, count, splits;
    __device__ __forceinline__ Entries(const Kv4Shared& a) {
        const int l = threadIdx.x & 63;
        first = a.gfirst[l]; part = a.gpart[l]; len = a.glen[l]; tile = a.gtile[l];
        lane = a.glane[l]; start = a.gstart[l]; count = a.gcount[l]; splits = a.gsplits[l];
    }
};
__device__ __forceinline__ int pick(int v, int j) { return __builtin_amdgcn_readlane(v, j); }
__device__ __forceinline__ int low16(uint2 v, int i) { return entry(v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16, i); }

// NQP, NQO: 16 rows a block takes of a prompt's and a wave of an answer's own.
// Long prompts are bound by instructions: 256 answers x 8 heads over 32,768 slots of 256 dims (69 GFLOP) 81.5 us a call with its
// join, 0.85 PFLOP/s; an MFMA has 5 other vector instructions beside it (codes and weights into bf16, exponentials), the SIMDs issue in 68 %
// of the busy cycles and the MFMA pipes work in 43 %. Without turning codes into bf16 it takes 8 us less; from which
// level of the memory the tiles come makes no difference, nor do loads further ahead. Shorter ones are bound by what surrounds the
// walk: over 4,096 slots 23.5 us, of which 11 are launch, Q, a first tile and the waves' join, 3.5 the partial results' stores.
// 128 dims: in the registers of three waves a SIMD, so that answers' blocks run beside two prompts' of a CU (8 x 32 answers over 8192
// slots 45.4 -> 42.5 us, a few registers spilled).
template <int D, int NQP, int NQO>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 3) shared_kernel(Kv4Shared a) {
    __shared__ Exchange<D> ex;
    static_assert(NQO == 1 || sizeof(ex.os) >= 4 * NQO * (D / 32) * 1024, "the waves' Q operands lie where their sums go at the end");
    const int per = a.T * (a.q_heads / a.kv_heads), lane = threadIdx.x & 63;
    const uint32_t seqs = ((const uint32_t*)a.seq)[lane];
    Part p;
    if ((int)blockIdx.x < a.prompt_blocks) {
        const Entries en(a);
        const int j = __popcll(__ballot(en.first <= (int)blockIdx.x)) - 1;
        const int len = pick(en.len, j), splits = pick(en.splits, j), tiles = (len + 31) >> 5;
        // splits vary fastest: the blocks of one split of a prompt, which read the same tiles, lie on one XCD where the
        // splits are a multiple of 8
        const uint32_t ix = blockIdx.x - pick(en.first, j), item = ix / (uint32_t)splits, split = ix - item * splits;
        const int each = (uint32_t)tiles / (uint32_t)splits, more = tiles - each * splits, rt = over(item, a.kv_inv);
        p.start = pick(en.start, j);
        p.rows = pick(en.count, j) * per;
        p.h = item - rt * a.kv_heads;
        p.rho0 = rt * NQP * 16;
        p.t0 = split * each + min((int)split, more);
        p.t1 = p.t0 + each + ((int)split < more);
        p.region = a.prefix + pick(en.lane, j) * a.prefix_lane + p.h * a.prefix_region;
        p.last = len - 1;
        p.pos = 0;
        p.tile = pick(en.part, j) + (split * a.kv_heads + p.h) * ((p.rows + 15) >> 4) + rt * NQP;
        part_rows<D, NQP, 4>(a, p, seqs, ex);
        return;
    }
    // Of a sequence's own slots a wave has a part to itself: the lists are short, and four waves of a block on one of them
    // took longer to join than to walk it.
    const int unit = __builtin_amdgcn_readfirstlane((blockIdx.x - a.prompt_blocks) * 4 + (threadIdx.x >> 6));
    if (unit >= a.own_units) return;
    const uint2 f = ((const uint2*)a.first)[lane], lanes = ((const uint2*)a.lane)[lane];
    const uint4 ps = ((const uint4*)a.pos)[lane];
    const int row_tiles = (per + NQO * 16 - 1) / (NQO * 16), zr = over(unit, a.kv_inv), z = (uint32_t)zr / (uint32_t)row_tiles, rt = zr - z * row_tiles;
    const uint32_t zz = (uint32_t)z;
    const int i = __popcll(__ballot((f.x & 0xffffu) <= zz)) + __popcll(__ballot((f.x >> 16) <= zz)) +
                  __popcll(__ballot((f.y & 0xffffu) <= zz)) + __popcll(__ballot((f.y >> 16) <= zz)) - 1;
    const int first = low16(f, i), splits = (i + 1 < a.n ? low16(f, i + 1) : a.own_splits) - first, split = z - first;
    p.start = i;
    p.rows = per;
    p.h = unit - zr * a.kv_heads;
    p.rho0 = rt * NQO * 16;
    p.pos = entry(ps.x, ps.y, ps.z, ps.w, i);
    const int tiles = ((p.pos + over(min(p.rho0 + NQO * 16, per) - 1, a.group_inv)) >> 5) + 1;
    const int each = (uint32_t)tiles / (uint32_t)splits, more = tiles - each * splits;
    p.t0 = split * each + min(split, more);
    p.t1 = p.t0 + each + (split < more);
    p.region = a.cache + low16(lanes, i) * a.lane_bytes + p.h * a.region;
    p.last = -1;
    p.tile = a.own_part + (z * a.kv_heads + p.h) * ((per + 15) >> 4) + rt * NQO;
    part_rows<D, NQO, 1>(a, p, seqs, ex);
}

// Answers with prompts too short to share: a block takes all that 16 or 32 rows of one see, and ends it.
template <int D, int NQ>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 3) whole_kernel(Kv4Shared a) {
    __shared__ Exchange<D> ex;
    const int per = a.T * (a.q_heads / a.kv_heads), lane = threadIdx.x & 63;
    const uint32_t seqs = ((const uint32_t*)a.seq)[lane];
    const uint2 lanes = ((const uint2*)a.lane)[lane];
    const uint4 ps = ((const uint4*)a.pos)[lane];
    const Entries en(a);
    const int row_tiles = (per + NQ * 16 - 1) / (NQ * 16), zr = over(blockIdx.x, a.kv_inv), i = (uint32_t)zr / (uint32_t)row_tiles;
    const int j = __popcll(__ballot(en.start <= i)) - 1;
    Part p;
    p.start = i;
    p.rows = per;
    p.h = blockIdx.x - zr * a.kv_heads;
    p.rho0 = (zr - i * row_tiles) * NQ * 16;
    p.len = pick(en.len, j);
    p.ahead = (p.len + 31) >> 5;
    p.prefix = a.prefix + pick(en.lane, j) * a.prefix_lane + p.h * a.prefix_region;
    p.region = a.cache + low16(lanes, i) * a.lane_bytes + p.h * a.region;
    p.last = -1;
    p.pos = entry(ps.x, ps.y, ps.z, ps.w, i);
    p.t0 = 0;
    p.t1 = p.ahead + ((p.pos + over(min(p.rho0 + NQ * 16, per) - 1, a.group_inv)) >> 5) + 1;
    p.tile = 0;
    part_rows<D, NQ, 4, true>(a, p, seqs, ex);
}

// Joins the parts of 16 rows of an entry. A wave takes one of a lane's runs of 4 dims (256 dims, so that there are waves enough)
// or its four of 1 or 2 (8192 rows of 128 dims: 9.8 us by 2 dims a lane, 7.3 by 8), some parts in flight. FEW rows of many
// parts: a block's eight waves take a run's parts in turn, and the first ends it (4 rows' 53 parts of 128 dims 22.6 -> 4.4 us;
// 1024 rows' 4 of 256 5.9 -> 15.2).
template <int D, bool FEW>
constexpr int kJoinBlocks = FEW ? 16 : D == 256 ? 4 : 1;     // for 16 rows
template <bool FEW>
constexpr int kJoinWaves = FEW ? 8 : 4;
template <int D, bool FEW>
__global__ void __launch_bounds__(64 * kJoinWaves<FEW>) shared_join(Kv4Shared a) {
    constexpr int N = kRun<D>, B = kJoinBlocks<D, FEW>, R = B == 1 ? 4 : 1, kJoin = B == 1 ? 4 : 8, W = FEW ? 8 : 1;
    __shared__ float states[FEW ? W : 1][R * N + 2][64];
    const int group = a.q_heads / a.kv_heads, per = a.T * group, lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t seqs = ((const uint32_t*)a.seq)[lane];
    const uint2 f = ((const uint2*)a.first)[lane];
    const Entries en(a);
    const int wv = threadIdx.x >> 6, r = B == 1 ? wv : blockIdx.x & 3, w0 = FEW ? blockIdx.x >> 2 & 3 : B == 1 ? 0 : wv, ix = blockIdx.x / B, j = __popcll(__ballot(en.tile <= ix)) - 1;
    const int start = pick(en.start, j), rows = pick(en.count, j) * per, tiles = (rows + 15) >> 4, part = pick(en.part, j);
    const int prompt = pick(en.len, j) ? pick(en.splits, j) : 0;
    const uint32_t it = ix - pick(en.tile, j);
    const int rt = over(it, a.kv_inv), h = it - rt * a.kv_heads, rho = rt * 16 + (lane & 15);
    // this lane's row: of sequence i its row s
    const int i0 = over(min(rho, rows - 1), a.per_inv), s = min(rho, rows - 1) - i0 * per, i = start + i0, t = over(s, a.group_inv);
    const int seq = __shfl((int)seqs, i >> 2) >> 8 * (i & 3) & 255;
    const auto first_of = [&](int k) {
        const int x = __shfl((int)f.x, k >> 2), y = __shfl((int)f.y, k >> 2), v = k & 2 ? y : x;
        return (k & 1 ? v >> 16 : v) & 0xffff;
    };
    const int first = first_of(i), next = first_of(min(i + 1, kSeqArgs - 1));
    const int own = (i + 1 < a.n ? next : a.own_splits) - first, own_tiles = (per + 15) >> 4;
    if (!FEW && rho >= rows) return;
    const int at = (64 * (4 * w0 + r) + 16 * g) * N;
    const float* pp = a.part + (size_t)(part + h * tiles + rt) * tile_floats(D);
    const float* po = a.part + (size_t)(a.own_part + (first * a.kv_heads + h) * own_tiles + (s >> 4)) * tile_floats(D);
    const size_t step = (size_t)a.kv_heads * tiles * tile_floats(D), own_step = (size_t)a.kv_heads * own_tiles * tile_floats(D);
    const int parts = prompt + own;
    float x[R * N], m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int e = 0; e < R * N; ++e) x[e] = 0.f;
    for (int k0 = FEW ? wv : 0; k0 < parts; k0 += W * kJoin) {
        float o[kJoin][R * N];
        float2 ml[kJoin];
#pragma unroll
        for (int k = 0; k < kJoin; ++k) {
            const int kk = min(k0 + W * k, parts - 1), n = kk < prompt ? lane & 15 : s & 15;
            const float* from = kk < prompt ? pp + kk * step : po + (kk - prompt) * own_step;
#pragma unroll
            for (int w = 0; w < R; ++w) __builtin_memcpy(&o[k][w * N], from + at + (256 * w + n) * N, 4 * N);
            ml[k] = *(const float2*)(from + 16 * D + 2 * n);
        }
        float mn = m;
#pragma unroll
        for (int k = 0; k < kJoin; ++k) mn = fmaxf(mn, ml[k].x);
        const float mz = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - mz);
        m = mn;
        sum *= al;
#pragma unroll
        for (int e = 0; e < R * N; ++e) x[e] *= al;
#pragma unroll
        for (int k = 0; k < kJoin; ++k) {
            if (k0 + W * k >= parts) break;
            const float c = __builtin_amdgcn_exp2f(ml[k].x - mz);
            sum += c * ml[k].y;
#pragma unroll
            for (int e = 0; e < R * N; ++e) x[e] += c * o[k][e];
        }
    }
    if constexpr (FEW) {
        states[wv][R * N][lane] = m;
        states[wv][R * N + 1][lane] = sum;
#pragma unroll
        for (int e = 0; e < R * N; ++e) states[wv][e][lane] = x[e];
        __syncthreads();
        if (wv || rho >= rows) return;
        float mn = m, f[W];
#pragma unroll
        for (int w = 1; w < W; ++w) mn = fmaxf(mn, states[w][R * N][lane]);
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < R * N; ++e) x[e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            f[w] = __builtin_amdgcn_exp2f(states[w][R * N][lane] - (mn == -INFINITY ? 0.f : mn));
            sum += f[w] * states[w][R * N + 1][lane];
#pragma unroll
            for (int e = 0; e < R * N; ++e) x[e] += f[w] * states[w][e][lane];
        }
    }
    Out(a, (long long)seq * a.TT + t, h * group + s - t * group).template store<R * N>(a, x, sum, (4 * g + r) * (D / 16) + w0 * N);
}

// Of one list, after the rules below: few sequences with few kv heads leave most CUs idle over a long one. An answer of 5 heads
// over one kv head to 32,768 slots has 64 blocks and takes 12.8 us; over as many slots of its own it has 64 waves, 17.3 us, where
// the attention of single lanes takes 12.3 (2 kv heads of 256 dims 21.7 and 14.1).
constexpr int kPromptSplits = 64, kOwnSplits = 64;
template <int D>
static hipError_t launch(Kv4Shared& a, hipStream_t st) {
    const int group = a.q_heads / a.kv_heads, per = a.T * group, nqo = per > 16 ? 2 : 1;
    int widest = per;
    for (int j = 0; j < a.entries; ++j) {
        a.gcount[j] = (uint16_t)((j + 1 < a.entries ? a.gstart[j + 1] : a.n) - a.gstart[j]);
        if (a.glen[j]) widest = std::max(widest, a.gcount[j] * per);
    }
    const int nqp = widest > 16 ? 2 : 1;
    const auto items = [&](int j) { return a.kv_heads * ((kv4_tiles(a.gcount[j] * per) + nqp - 1) / nqp); };
    const auto prompt_tiles = [&](int j) { return (a.glen[j] + 31) >> 5; };
    const auto own_tiles = [&](int i) { return ((a.pos[i] + a.T - 1) >> 5) + 1; };
    const long long own_items = a.kv_heads * ((kv4_tiles(per) + nqo - 1) / nqo);
    a.per_inv = reciprocal(per);
    a.group_inv = reciprocal(group);
    a.kv_inv = reciprocal(a.kv_heads);
    for (int j = a.entries; j < kEntryArgs; ++j) {
        a.gfirst[j] = a.gtile[j] = INT_MAX;
        a.gstart[j] = 0xffff;
    }
    long long work = 0, own = 0, steps = 0, longest = 0, part = 0, blocks = 0, joins = 0;
    for (int j = 0; j < a.entries; ++j) {
        work += prompt_tiles(j) * items(j);
        a.gtile[j] = (int)joins;
        joins += a.kv_heads * kv4_tiles(a.gcount[j] * per);
        for (int i = a.gstart[j]; i < a.gstart[j] + a.gcount[j]; ++i) {
            own += own_tiles(i) * own_items;
            steps += (prompt_tiles(j) + own_tiles(i)) * own_items;
            longest = std::max<long long>(longest, prompt_tiles(j) + own_tiles(i));
        }
    }
    // Short lists are walked whole, without parts and their join, some 4 us less: while a wave's quarter of the longest takes
    // no more than 7 us (a tile 0.7, 0.4 and 0.33 us of 256, 128 and 64 dims, half as much again for 32 rows), and all
    // of them not much more than with the prompts shared (4 us are 13,000 tiles on the card); longer ones where sharing saves
    // little, and there are so many that the longest one's end does not matter. Calls, us, in parts and whole: 12.9 and 8.5 for 6
    // answers to 4 slots, 15.7 and 11.9 for 143 to 246, 18.5 and 10.9 for 2 x 29 x 2 rows to 234 with 615 of their own, 101 and 68
    // for 6 x 27 x 3 rows to 1281 with 505 of their own; 12.9 and 16.6 for 2 x 11 to 2091, 20.5 and 35.6 for 135 x 3 rows to 1400.
    // Over 390 drawn cases the geometric mean is within 1 % of the better form's; seven cases miss it by more than a tenth, six
    // lists of 47 to 107 tiles in parts (41 x 3 rows to 1175 with 506 of their own, 48 / 3 heads of 256: 34.5 for 25.7) and one
    // of 96 whole (8 to 3019, 16 heads of 64: 16.2 for 12.7).
    const long long shared = work + own, most = (long long)(28 / (0.2 + D / 512.0) / (nqo == 2 ? 1.5 : 1.0));
    const bool whole = longest < 1 << 25 &&         // (their slots are numbered in one row)
                       ((longest <= most && steps <= 2 * shared + 13000) || (steps * 5 <= shared * 7 && longest * 300 <= steps));
    if (whole) {
        hipLaunchKernelGGL((nqo == 1 ? whole_kernel<D, 1> : whole_kernel<D, 2>), dim3((unsigned)(a.n * own_items)), dim3(256), 0, st, a);
        return hipGetLastError();
    }
    // One block a CU, or two where each has 128 tiles or more: a second wave on a SIMD fills the waits of the first (512
    // tiles of 256 dims: 97.8 -> 83.3 us; about 160 of 128: 56.6 -> 42.5), but twice the partial results take their time to write
    // and to join (64 tiles of 256 dims: 23.8 + 5.7 -> 29.7 + 7.8). No block more than that, which would run behind them,
    // and 16 tiles at least (64 answers x 3 rows x 2000 slots, 48 items of 63 tiles: 12 tiles in 288 blocks 19.6 + 5.8, 16
    // in 192 16.2 + 5.1).
    const auto prompt_blocks = [&](long long tiles) {
        long long s = 0;
        for (int j = 0; j < a.entries; ++j) s += (prompt_tiles(j) + tiles - 1) / tiles * items(j);
        return s;
    };
    const long long most_blocks = (work + 255) / 256 < 128 ? 256 : 512;
    // Few rows, whose parts' join takes them by eight waves: down to 4 tiles in no more than 128 blocks (8 answers to 3000 slots
    // of 256 dims 12.1 -> 8.7 us, 32 to 8000 in 256 blocks of 8 tiles 16.0, in 128 of 16 14.1), an answer's own by 4 (one
    // of 7000 11.4 -> 8.1).
    const bool few = joins <= 32, short_blocks = few && work < 128 * 16;
    long long tiles = short_blocks ? std::max<long long>(4, (work + 127) / 128) : std::max<long long>(16, (work + most_blocks - 1) / most_blocks);
    const long long least_blocks = prompt_blocks(INT_MAX);
    while (prompt_blocks(tiles) > std::max(most_blocks, least_blocks)) tiles += (tiles + 7) / 8;
    int parts = 0;                   // of a row, at most
    long long own_per = std::max<long long>(few ? 4 : 8, (own + 2047) / 2048);
    for (;; tiles *= 2, own_per *= 2) {
        part = blocks = 0;
        int from_prompt = 0, from_own = 0;
        bool least = true;
        for (int j = 0; j < a.entries; ++j) {
            const int s = (int)std::min<long long>(kPromptSplits, (prompt_tiles(j) + tiles - 1) / tiles);
            least &= s <= 1;
            a.gfirst[j] = (int)blocks;
            a.gpart[j] = (int)part;
            a.gsplits[j] = (uint16_t)std::max(1, s);
            blocks += s * items(j);
            from_prompt = std::max(from_prompt, s);
            part += s * a.kv_heads * kv4_tiles(a.gcount[j] * per);
        }
        a.prompt_blocks = (int)blocks;
        a.own_part = (int)part;
        int z = 0;
        for (int i = 0; i < a.n; ++i) {
            const int s = (int)std::min<long long>(kOwnSplits, (own_tiles(i) + own_per - 1) / own_per);
            least &= s == 1;
            a.first[i] = (uint16_t)z;
            z += s;
            from_own = std::max(from_own, s);
        }
        a.own_splits = z;
        a.own_units = (int)(z * own_items);
        part += z * a.kv_heads * kv4_tiles(per);
        blocks += (a.own_units + 3) / 4;
        parts = from_prompt + from_own;
        if (part <= kv4_shared_room(D) || least) break;
    }
    for (int i = a.n; i < kSeqArgs; ++i) a.first[i] = 0xffff;
    if (part > kv4_shared_room(D) || blocks > kLaunchBlocks || joins * 16 > kLaunchBlocks) return hipErrorInvalidValue;
    const auto k = nqp == 1 ? shared_kernel<D, 1, 1> : nqo == 1 ? shared_kernel<D, 2, 1> : shared_kernel<D, 2, 2>;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, a);
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    if (joins <= std::max(32, 2 * parts))          // (288 rows' 8 parts, 36 of these, 5.7 -> 7.7)
        hipLaunchKernelGGL((shared_join<D, true>), dim3((unsigned)joins * kJoinBlocks<D, true>), dim3(64 * kJoinWaves<true>), 0, st, a);
    else
        hipLaunchKernelGGL((shared_join<D, false>), dim3((unsigned)joins * kJoinBlocks<D, false>), dim3(64 * kJoinWaves<false>), 0, st, a);
    return hipGetLastError();
}
hipError_t launch_attn_kv4_shared(Kv4Shared& a, hipStream_t st) {
    return a.D == 256 ? launch<256>(a, st) : a.D == 128 ? launch<128>(a, st) : launch<64>(a, st);
}

}  // namespace q35
