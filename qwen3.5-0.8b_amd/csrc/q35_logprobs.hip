// Log probabilities of given tokens, their ranks, the rows' entropy and most likely tokens, in one pass over the logits
// (in two where ties or masks leave too many tokens that may be among the most likely).
//
// With z_i = (x_i - m) / T, m = max x, S = sum e^z_i, A = sum z_i e^z_i of a row:
//   log p_i = z_i - log S,   entropy = log S - A / S,   rank of t = #{x_i > x_t} + #{x_i = x_t, i < t},
// and the most likely tokens are the first of the order (x falling, i rising). Both sums move with m by a
// factor (and A by a multiple of S), so every wave keeps its own m and the states are joined at the end.
// A token that is all but certain has log p ~ -(S - 1): there the term 1 of the maximum itself goes into a float64
// sum by itself, so that S - 1 keeps float32's relative accuracy and does not end at 2^-24.
#include <algorithm>
#include <type_traits>

#include "q35_answers.h"
#include "q35_common.h"

namespace q35 {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// What a row's block leaves: the state of its sums (log2 units: z2 = (x - m) c) and its best tokens.
struct LpPart {
    double s, a;
    float m;
    int above;                       // tokens before the target in the order
};
constexpr int kParts = 64;           // blocks of one row, at most
constexpr int kPartRooms = 8192;     // (row, block)s of one launch
size_t logprob_ws_bytes() { return kPartRooms * (sizeof(LpPart) + kTopMost * sizeof(float2)); }

template <int CTRL>
__device__ __forceinline__ double move_d(double v) {
    const unsigned long long w = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)w, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(w >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum_d(double v) {
    v += move_d<0x128>(v);
    v += move_d<0x124>(v);
    v += move_d<0x4E>(v);
    v += move_d<0xB1>(v);
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) { return (a > b) | ((a == b) & (ia < ib)); }
__device__ __forceinline__ bool before(float2 a, float2 b) { return before(a.x, __float_as_int(a.y), b.x, __float_as_int(b.y)); }
__device__ __forceinline__ float2 nobody() { return make_float2(-INFINITY, __int_as_float(0x7fffffff)); }
// How many of list[0 .. n) come before mine. Eight at a time, past n too: there lie nobody()s.
constexpr int kPad = 8;
__device__ __forceinline__ int rank_in(const float2* list, int n, float2 mine) {
    int r = 0;
    for (int k = 0; k < n; k += kPad) {
        float2 o[kPad];
#pragma unroll
        for (int i = 0; i < kPad; ++i) o[i] = list[k + i];
#pragma unroll
        for (int i = 0; i < kPad; ++i) r += before(o[i], mine);
    }
    return r;
}

// A floor that at least `top` of the lanes' numbers reach: the smallest that fewer than `top` exceed.
__device__ __forceinline__ float floor_of(float x, int top) {
    int r = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) r += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__float_as_int(x), i)) > x;
    return -wave_max(r < top ? -x : -INFINITY);
}

// The running sums of a wave's lanes, all against the same m.
struct Sums { float m; double s, a; };
__device__ __forceinline__ void raise(Sums& u, float m, float c) {     // m > u.m, the same in every lane
    if (u.m > -INFINITY) {
        const float z = (u.m - m) * c, f = __builtin_amdgcn_exp2f(z);
        u.a = f > 0.f ? f * (u.a + z * u.s) : 0.0;
        u.s *= f;
    }
    u.m = m;
}

// A row's results but its best tokens.
__device__ __forceinline__ void finish(const LogprobArgs& a, int row, const LpPart& p, bool bad, double lse) {
    const int t = a.targets ? a.targets[row] : -1;
    const bool on = !bad && t >= 0 && t < a.vocab;
    if (a.logprobs) {
        double v = NAN;
        if (on) {
            const long long i = row * a.ld + t;
            const float x = a.bf16 ? bf2f(((const uint16_t*)a.logits)[i]) : ((const float*)a.logits)[i];
            v = (((double)x - p.m) * a.c - lse) * 0.69314718055994530942;
        }
        a.logprobs[row] = (float)v;
    }
    if (a.ranks) a.ranks[row] = on ? p.above : -1;
    if (a.entropy) a.entropy[row] = bad ? NAN : (float)((lse - p.a / p.s) * 0.69314718055994530942);
}
__device__ __forceinline__ bool no_distribution(const LpPart& p) { return !(p.s > 0.0) || !(p.s < INFINITY) || !(p.m < INFINITY); }
__device__ __forceinline__ void store_top(const LogprobArgs& a, int row, int r, float2 token, bool bad, float m, double lse) {
    const long long o = (long long)row * a.top + r;
    if (a.top_ids) a.top_ids[o] = bad ? -1 : __float_as_int(token.y);
    if (a.top_logprobs)
        a.top_logprobs[o] = bad ? NAN : (float)((((double)token.x - m) * a.c - lse) * 0.69314718055994530942);
}
// A part's state against the common m.
__device__ __forceinline__ void against(const LpPart& q, float m, double c, double& s, double& a) {
    s = a = 0.0;
    if (q.m == -INFINITY && q.s == 0.0) return;
    const double z = q.m == m ? 0.0 : ((double)q.m - m) * c, f = exp2(z);
    s = f * q.s;
    a = f > 0.0 ? f * (q.a + z * q.s) : 0.0;
}

__device__ __forceinline__ float eight(const float* w) {
    return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
}
constexpr int kEach = 32;            // elements of a lane's tile
template <bool BF16>
__device__ __forceinline__ float element(const u32x4* w, int i) {
    if (BF16) {
        const uint32_t v = w[i / 8][i % 8 / 2];
        return __uint_as_float(i % 2 ? v & 0xffff0000u : v << 16);
    }
    return __uint_as_float(w[i / 4][i % 4]);
}

// The best tokens of a wave: a list of (logit, id) in LDS that holds every token it has met that may be among
// the row's `top` first, and at most kTight of them after each step. floor: what a token's logit must reach
// (strict: exceed, since `top` tokens of lower ids reach it) to get in.
constexpr int kTight = 64, kStep = 512, kList = kTight + kStep;
struct Best {
    float2* list;                    // [kList + kPad]: logit, id as bits
    float2* sorted;                  // [kTopMost]
    float floor;
    bool strict;
    int count, top;
};
// Keeps the list's first `top` in order.
__device__ __forceinline__ void tighten(Best& b) {
    const int lane = threadIdx.x & 63;
    if (lane < kPad) b.list[b.count + lane] = nobody();
    wave_sync();
    for (int c = lane; c < b.count; c += 64) {
        const float2 mine = b.list[c];
        const int r = rank_in(b.list, b.count, mine);
        if (r < b.top) b.sorted[r] = mine;
    }
    wave_sync();
    b.count = min(b.count, b.top);
    if (lane < b.count) b.list[lane] = b.sorted[lane];
    wave_sync();
    if (b.count == b.top) {
        b.floor = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__float_as_int(b.sorted[b.top - 1].x)));
        b.strict = true;
    }
}
// One element a lane.
__device__ __forceinline__ void push(Best& b, float x, int id, bool on) {
    const bool in = on && (b.strict ? x > b.floor : x >= b.floor);
    const unsigned long long mask = __ballot(in);
    if (!mask) return;
    if (in) b.list[b.count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] =
        make_float2(x, __int_as_float(id));
    b.count += __popcll(mask);
}

// A block per (row, part of it). The row's 16-byte pieces go to waves in tiles of kEach elements a lane; the up to 14
// elements in front of its first whole piece and behind its last (edges) are the first part's first wave's. A row of one
// part is finished here, others by logprobs_join.
// The best tokens: while the sums are made, a lane keeps the largest of its elements of each run of tiles. Of those
// lanes the same ones of the waves make 64 groups; `top` groups reach the top-th largest of their
// maxima (floor), so the row's best do, and only the pieces of the lanes and runs that reach it are read
// again: some 25 of them for 20 tokens, of any number of elements. If ties or infinities bring more candidates than there is
// room for, the part is gone over in order with a list a wave (Best). Fewer than `top` groups with a finite logit have no
// floor, and every element is a candidate: masks that leave 10 tokens of a row take 1999 rows of 32,003 with 20 tokens
// from 52 to 128 us in float32 and from 35 to 236 in bfloat16, one row of 248,320 from 12.6 to 96 and from 12.9 to 176
// (256 rows of 248,320 with 5 tokens, fewer than those 10, take what they took).
// float32: bound by memory, 256 rows of 248,320 with 5 tokens each (254 MB) 51 us over buffers in turn, 5.0 TB/s (one buffer over
// and over, which the last cache nearly holds, 44 us). bfloat16: by memory and the 8 instructions an element takes here (the
// entropy's among them, also where it is not wanted), 1999 rows of 32,003 with 20 tokens (128 MB) 37 us, 3.5 TB/s (without
// tokens 31.8 of 37.4 on one buffer). One row of 248,320: a chain of loads and barriers, 8.8 us and the join's 3.8.
template <int W>
constexpr int kRuns = W > 4 ? 64 / W : 16;       // of a part's tiles a wave
template <int W>
constexpr int kRoom = W > 4 ? 64 * W : 256;      // candidates, and lanes' runs that may hold some; a list of kTight a wave
template <bool BF16, bool TOP, int W>
__global__ void __launch_bounds__(64 * W, W > 4 ? 4 : 5) logprobs_kernel(LogprobArgs a, int row0) {
    constexpr int V = BF16 ? 8 : 4, L = kEach / V;
    struct Lists { float2 list[W][kList + kPad], sorted[W][kTopMost]; };
    union Store {
        float runs[kRuns<W>][64 * W];
        Lists lists;
    };
    __shared__ __align__(16) char store[TOP ? sizeof(Store) : 16];
    Store* st = (Store*)store;
    __shared__ float2 flat[TOP ? kRoom<W> + kPad : 1];
    __shared__ uint16_t held[TOP ? kRoom<W> : 1];
    __shared__ LpPart waves[W];
    __shared__ int counts[W], n_held, n_flat;
    __shared__ double row_lse;
    __shared__ float row_m, row_floor;
    const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63;
    const int part = blockIdx.x % a.parts, row = row0 + blockIdx.x / a.parts;
    const char* base = (const char*)a.logits + row * a.ld * (BF16 ? 2 : 4);
    const int head = min((int)((16 - ((uintptr_t)base & 15)) & 15) / (BF16 ? 2 : 4), a.vocab);
    const int pieces = (a.vocab - head) / V, tiles = (pieces + 64 * L - 1) / (64 * L);
    const int t0 = (int)((long long)tiles * part / a.parts), t1 = (int)((long long)tiles * (part + 1) / a.parts);
    const char* body = base + head * (BF16 ? 2 : 4);
    const uint32_t none = BF16 ? 0xff80ff80u : 0xff800000u;
    const auto fetch = [&](u32x4* buf, int t) {
        if ((t + 1) * L * 64 <= pieces) {
            const char* from = body + (size_t)t * (L * 1024);
#pragma unroll
            for (int i = 0; i < L; ++i) buf[i] = *(const u32x4*)(from + lane * 16 + i * 1024);
            return;
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int p = (t * L + i) * 64 + lane;
            buf[i] = u32x4{none, none, none, none};
            if (p < pieces) buf[i] = *(const u32x4*)(body + (size_t)p * 16);
        }
    };
    const auto at = [&](int i) {
        return BF16 ? __uint_as_float((uint32_t)((const uint16_t*)base)[i] << 16) : ((const float*)base)[i];
    };
    int target = a.targets ? a.targets[row] : -1;
    u32x4 buf[L];
    if (t0 + wv < t1) fetch(buf, t0 + wv);
    if (target >= a.vocab) target = -1;
    // Tokens before the target: of the pieces before its own those that reach x_t, of the others those that reach the
    // next float32 above it, and in its own piece (tp) the lower ids with x_t as well.
    const float xt = target >= 0 ? at(target) : INFINITY;
    const uint32_t tb = __float_as_uint(xt);
    const float over = __uint_as_float(xt == 0.f ? 1u : tb >> 31 ? tb - 1u : tb + 1u);
    const int tp = target < head ? -1 : min((target - head) / V, pieces);
    const float c = (float)a.c;
    Sums u = {-INFINITY, 0.0, 0.0};
    int above = 0;
    // the edges: an element a lane
    const int tail = head + pieces * V, edge = lane < head ? lane : tail + lane - head;
    const bool edges = part == 0 && wv == 0, on_edge = edges && edge < a.vocab;
    const float x_edge = on_edge ? at(edge) : -INFINITY;
    if (edges) {
        const float top = wave_max(x_edge);
        if (top > u.m) raise(u, top, c);
        const float z = on_edge ? (x_edge - (u.m == -INFINITY ? 0.f : u.m)) * c : -INFINITY, w = __builtin_amdgcn_exp2f(z);
        u.s += w;
        u.a += w * __builtin_elementwise_maximum(z, -200.f);
        above += __popcll(__ballot(on_edge && before(x_edge, edge, xt, target)));
        if (tp >= 0 && tp < pieces) {
            const int id = head + tp * V + lane;
            above += __popcll(__ballot(id < target && at(min(id, target)) == xt));
        }
    }
    const int each = (t1 - t0 + W * kRuns<W> - 1) / (W * kRuns<W>);       // tiles of a run
    float run = -INFINITY;
    int n_run = 0, i_run = 0, t_max = -1;
    for (int t = t0 + wv; t < t1; t += W) {
        float x[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = element<BF16>(buf, i);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
        if (__any(top > u.m)) {
            raise(u, wave_max(fmaxf(top, u.m)), c);
            t_max = t;
        }
        const float m = u.m == -INFINITY ? 0.f : u.m;
        // float32 sums of eight terms by halves, then of the four eights: 5 roundings each
        float ss = 0.f, as = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; i += 8) {
            float w[8], z[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                z[k] = (x[i + k] - m) * c;
                w[k] = __builtin_amdgcn_exp2f(z[k]);
                as = __builtin_fmaf(w[k], __builtin_elementwise_maximum(z[k], -200.f), as);
            }
            ss += eight(w);
            asm volatile("" : "+v"(as), "+v"(ss));   // now: or all 32 terms wait for a later place, in 64 registers
        }
        u.a += as;
        u.s += ss;
        if (__any(top >= xt)) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const float reach = (t * L + i) * 64 + lane < tp ? xt : over;
#pragma unroll
                for (int k = 0; k < V; ++k) n += __popcll(__ballot(x[i * V + k] >= reach));
            }
            above += n;
        }
        if (TOP) {
            run = fmaxf(run, top);
            if (++n_run == each) {
                st[0].runs[i_run++][tid] = run;
                run = -INFINITY;
                n_run = 0;
            }
        }
        if (t + W < t1) fetch(buf, t + W);
    }
    double s = wave_sum_d(u.s);
    if (t_max >= 0 && s < 2.0 && u.m < INFINITY) {
        // the maximum all but alone: its tile's float32 sums again, with its 1 apart from the rest
        fetch(buf, t_max);
        float ss = 0.f, rest = 0.f;
        int ones = 0;
#pragma unroll
        for (int i = 0; i < kEach; i += 8) {
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = __builtin_amdgcn_exp2f((element<BF16>(buf, i + k) - u.m) * c);
            ss += eight(w);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (element<BF16>(buf, i + k) == u.m) { ++ones; w[k] = 0.f; }
            rest += eight(w);
        }
        s = wave_sum_d(u.s - ss + rest + ones);
    }
    u.s = s;
    u.a = wave_sum_d(u.a);
    if (lane == 0) waves[wv] = {u.s, u.a, u.m, above};
    if (TOP) {
        for (; i_run < kRuns<W>; ++i_run, run = -INFINITY) st[0].runs[i_run][tid] = run;
        if (tid == 0) n_held = n_flat = 0;
    }
    __syncthreads();
    const size_t room = blockIdx.x;
    if (wv == W - 1) {
        LpPart p = lane < W ? waves[lane] : LpPart{0.0, 0.0, -INFINITY, 0};
        const float m = wave_max(p.m);
        double s, e;
        against(p, m, a.c, s, e);
        p = {wave_sum_d(s), wave_sum_d(e), m, (int)wave_sum_d(p.above)};
        if (lane == 0) {
            if (a.parts == 1) {
                const bool bad = no_distribution(p);
                const double l = bad ? (double)NAN : log2(p.s);
                row_lse = l;
                row_m = m;
                finish(a, row, p, bad, l);
            } else {
                ((LpPart*)a.ws)[room] = p;
            }
        }
    }
    if (!TOP) return;
    if (wv == 0) {
        float most = -INFINITY;
#pragma unroll
        for (int r = 0; r < kRuns<W>; ++r)
#pragma unroll
            for (int w = 0; w < W; ++w) most = fmaxf(most, st[0].runs[r][w * 64 + lane]);
        const float f = floor_of(most, a.top);
        if (lane == 0) row_floor = f;
    }
    __syncthreads();
    const float floor = row_floor;
    for (int r = 0; r < kRuns<W>; ++r) {
        const int t = t0 + wv + W * r * each;        // the run's first tile
        if (t < t1 && t * L * 64 + lane < pieces && st[0].runs[r][tid] >= floor) {
            const int k = atomicAdd(&n_held, 1);
            if (k < kRoom<W>) held[k] = (uint16_t)(r * 64 * W + tid);
        }
    }
    __syncthreads();
    const int runs = n_held;
    if (runs <= kRoom<W>) {
        const auto keep = [&](float x, int id) {
            if (!(x >= floor)) return;
            const int k = atomicAdd(&n_flat, 1);
            if (k < kRoom<W>) flat[k] = make_float2(x, __int_as_float(id));
        };
        if (on_edge) keep(x_edge, edge);
        for (int i = tid; i < runs * each * L; i += 64 * W) {
            const int h = held[i / (each * L)], k = i % (each * L);
            const int t = t0 + h / 64 % W + W * (h / (64 * W) * each + k / L), p = (t * L + k % L) * 64 + h % 64;
            if (t >= t1 || p >= pieces) continue;
            const u32x4 w = *(const u32x4*)(body + (size_t)p * 16);
#pragma unroll
            for (int e = 0; e < V; ++e) keep(element<BF16>(&w, e), head + p * V + e);
        }
    }
    __syncthreads();
    int all = n_flat;
    if (runs > kRoom<W> || all > kRoom<W>) {       // in order, a list a wave
        __syncthreads();                     // (st was read as runs, n_flat by all)
        Best best = {st[0].lists.list[wv], st[0].lists.sorted[wv], floor, false, 0, a.top};
        if (edges) push(best, x_edge, edge, on_edge && lane < head);
        for (int t = t0 + wv; t < t1; t += W) {
            fetch(buf, t);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int p = (t * L + i) * 64 + lane;
#pragma unroll
                for (int k = 0; k < V; ++k) push(best, element<BF16>(buf, i * V + k), head + p * V + k, p < pieces);
                if (best.count > kTight) tighten(best);
            }
        }
        if (edges) push(best, x_edge, edge, on_edge && lane >= head);
        if (best.count > kTight) tighten(best);
        if (lane == 0) counts[wv] = best.count;
        __syncthreads();
        int from = 0;
        all = 0;
        for (int w = 0; w < W; ++w) {
            if (w < wv) from += counts[w];
            all += counts[w];
        }
        if (lane < best.count) flat[from + lane] = best.list[lane];
    }
    if (tid < kPad) flat[all + tid] = nobody();
    __syncthreads();
    float2* tops = (float2*)(a.ws + kPartRooms * sizeof(LpPart)) + room * kTopMost;
    const bool bad = a.parts == 1 && row_lse != row_lse;
    for (int i = tid; i < all && !bad; i += 64 * W) {
        const int r = rank_in(flat, all, flat[i]);
        if (r >= a.top) continue;
        if (a.parts > 1) tops[r] = flat[i];
        else store_top(a, row, r, flat[i], false, row_m, row_lse);
    }
    if (a.parts > 1 && tid >= all && tid < a.top) tops[tid] = nobody();
    if (bad && tid < a.top) store_top(a, row, tid, nobody(), true, 0.f, 0.0);
}

// Joins a row's parts: a block a row. Of the parts' sorted lists only what may be among the first `top` of all is ranked:
// what reaches the top-th largest of 64 of them, the parts' firsts, seconds and so on.
template <bool TOP>
__global__ void __launch_bounds__(256) logprobs_join(LogprobArgs a, int row0) {
    __shared__ float2 kept[TOP ? kParts * kTopMost + kPad : 1];
    __shared__ int count;
    __shared__ double lse;
    __shared__ float mx, least;
    const int tid = threadIdx.x, row = row0 + blockIdx.x;
    const LpPart* parts = (const LpPart*)a.ws + (size_t)blockIdx.x * a.parts;
    const float2* tops = (const float2*)(a.ws + kPartRooms * sizeof(LpPart)) + (size_t)blockIdx.x * a.parts * kTopMost;
    const int n = TOP ? a.parts * a.top : 0;
    float2 mine[kParts * kTopMost / 256];
    if (TOP) {
#pragma unroll
        for (int i = 0; i < kParts * kTopMost / 256; ++i) {
            const int k = tid + 256 * i;
            mine[i] = k < n ? tops[k / a.top * kTopMost + k % a.top] : nobody();
        }
    }
    if (tid < 64) {
        LpPart p = tid < a.parts ? parts[tid] : LpPart{0.0, 0.0, -INFINITY, 0};
        const float m = wave_max(p.m);
        double s, e;
        against(p, m, a.c, s, e);
        int above = p.above;
        for (int k = 32; k; k >>= 1) above += __shfl_xor(above, k);
        p = {wave_sum_d(s), wave_sum_d(e), m, above};
        if (tid == 0) {
            const bool bad = no_distribution(p);
            const double l = bad ? (double)NAN : log2(p.s);
            lse = l;
            mx = m;
            count = 0;
            finish(a, row, p, bad, l);
        }
    } else if (TOP && tid < 128) {
        const int i = tid - 64, depth = i / a.parts;
        const bool on = depth < min(64 / a.parts, a.top);
        const float f = floor_of(on ? tops[i % a.parts * kTopMost + depth].x : -INFINITY, a.top);
        if (tid == 64) least = f;
    }
    if (!TOP) return;
    __syncthreads();
    if (lse != lse) {
        if (tid < a.top) store_top(a, row, tid, nobody(), true, 0.f, 0.0);
        return;
    }
#pragma unroll
    for (int i = 0; i < kParts * kTopMost / 256; ++i)
        if (mine[i].x >= least && __float_as_int(mine[i].y) < a.vocab) kept[atomicAdd(&count, 1)] = mine[i];
    __syncthreads();
    const int all = count;
    if (tid < kPad) kept[all + tid] = nobody();
    __syncthreads();
    for (int k = tid; k < all; k += 256) {
        const int r = rank_in(kept, all, kept[k]);
        if (r < a.top) store_top(a, row, r, kept[k], false, mx, lse);
    }
}

hipError_t launch_logprobs(LogprobArgs a, hipStream_t st) {
    const int el = a.bf16 ? 8 : 4, tiles = (a.vocab / el + 64 * kEach / el - 1) / (64 * kEach / el);
    // A row is one block's where 512 rows or fewer have as many as tiles (of 2048 elements) at least: 16 waves up to 256
    // rows, a block a CU, and 8 above, two. Without a second launch and its join 256 rows of 248,320 float32 and 5 tokens take
    // 45.0 instead of 47.3 + 4.7 us (one buffer over and over), 16 of 32,003 bfloat16 and 20 tokens 11.6 for 9.5 + 4.5, 448 17 for 18 + 5; where rows
    // are fewer than tiles a CU takes too long for one (64 of 248,320 26.1 for 18.2 + 4.0; 75 of 151,936 even).
    // Otherwise blocks of four waves, as many of a row as give every CU four, each wave with a tile at least. The card holds
    // about 1280 of them: of more rows a block has two waves, whose ends fill the CUs better (1999 rows of 32,003 bf16 42.3 ->
    // 37.6 us).
    const bool whole = tiles > 4 && a.rows >= tiles && a.rows <= 512;
    const int waves = whole ? a.rows > 256 ? 8 : 16 : a.rows > 1280 ? 2 : 4;
    a.parts = whole ? 1 : std::max(1, std::min({kParts, (tiles + 3) / 4, 1024 / a.rows}));
    const int most = kPartRooms / a.parts;
    const auto pick = [&](auto bf16, auto top) {
        constexpr bool b = decltype(bf16)::value, t = decltype(top)::value;
        return waves == 16 ? logprobs_kernel<b, t, 16> : waves == 8 ? logprobs_kernel<b, t, 8> : waves == 4 ? logprobs_kernel<b, t, 4> : logprobs_kernel<b, t, 2>;
    };
    using Yes = std::true_type;
    using No = std::false_type;
    const auto k = a.bf16 ? (a.top ? pick(Yes{}, Yes{}) : pick(Yes{}, No{})) : (a.top ? pick(No{}, Yes{}) : pick(No{}, No{}));
    for (int r = 0, m; r < a.rows; r += m) {
        m = std::min(most, a.rows - r);
        hipLaunchKernelGGL(k, dim3((unsigned)(m * a.parts)), dim3(64 * waves), 0, st, a, r);
        hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
        if (a.parts == 1) continue;
        hipLaunchKernelGGL(a.top ? logprobs_join<true> : logprobs_join<false>, dim3(m), dim3(256), 0, st, a, r);
        rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

}  // namespace q35
