// Log probabilities of given tokens, their ranks, the rows' entropy and most likely tokens, in one pass over the logits.
//
// With z_i = (x_i - m) / T, m = max x, S = sum e^z_i, A = sum z_i e^z_i of a row:
//   log p_i = z_i - log S,   entropy = log S - A / S,   rank of t = #{x_i > x_t} + #{x_i = x_t, i < t},
// and the most likely tokens are the first of the order (x falling, i rising). Both sums move with m by a
// factor (and A by a multiple of S), so every wave keeps its own m and the states are joined at the end.
// A token that is all but certain has log p ~ -(S - 1): the term 1 of the maximum itself goes into a float64
// sum by itself, so that S - 1 keeps float32's relative accuracy and does not end at 2^-24.
#include <algorithm>

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

// The best tokens of a wave so far: a list of (logit, id) in LDS that holds every token it has met that may be among
// the row's `top` first, and at most kTight of them after each step. floor: what a token's logit must reach
// (strict: exceed, since `top` tokens of lower ids reach it) to get in.
constexpr int kTight = 64, kStep = 512, kList = kTight + kStep;
struct Best {
    float2* list;                    // [kList]: logit, id as bits
    float2* sorted;                  // [kTopMost]
    float floor;
    bool strict;
    int count, top;
};
__device__ __forceinline__ bool gets_in(const Best& b, float x) { return b.strict ? x > b.floor : x >= b.floor; }
// Keeps the list's first `top` in order.
__device__ __forceinline__ void tighten(Best& b) {
    const int lane = threadIdx.x & 63;
    wave_sync();
    for (int c = lane; c < b.count; c += 64) {
        const float2 mine = b.list[c];
        int r = 0;
        for (int k = 0; k < b.count; ++k) {
            const float2 o = b.list[k];
            r += before(o.x, __float_as_int(o.y), mine.x, __float_as_int(mine.y));
        }
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
    const bool in = on && gets_in(b, x);
    const unsigned long long mask = __ballot(in);
    if (!mask) return;
    if (in) b.list[b.count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] =
        make_float2(x, __int_as_float(id));
    b.count += __popcll(mask);
}
// The `top`-th largest of the lanes' maxima: a floor that `top` tokens reach at least.
__device__ __forceinline__ float floor_of(float x, int top) {
    const int lane = threadIdx.x & 63;
    int r = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__float_as_int(x), i));
        r += before(o, i, x, lane);
    }
    const unsigned long long at = __ballot(r == top - 1);
    if (!at) return -INFINITY;       // (a NaN among them)
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__float_as_int(x), __ffsll((long long)at) - 1));
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

constexpr int kLoads = 8;            // 16-byte loads of a lane's tile
template <bool BF16>
__device__ __forceinline__ float element(const u32x4* w, int i) {
    if (BF16) {
        const uint32_t v = w[i / 8][i % 8 / 2];
        return __uint_as_float(i % 2 ? v & 0xffff0000u : v << 16);
    }
    return __uint_as_float(w[i / 4][i % 4]);
}

// A block per (row, part of it). The row's 16-byte pieces go to waves in tiles of 64 x kLoads, the next tile's loads in
// flight; the up to 14 elements in front of its first whole piece and behind its last are the first part's first wave's.
template <bool BF16, bool TOP>
__global__ void __launch_bounds__(256) logprobs_kernel(LogprobArgs a, int row0) {
    constexpr int V = BF16 ? 8 : 4, E = kLoads * V;
    __shared__ float2 lists[TOP ? 4 : 1][TOP ? kList : 1], sorts[TOP ? 4 : 1][TOP ? kTopMost : 1];
    __shared__ LpPart waves[4];
    __shared__ int counts[4];
    const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63;
    const int part = blockIdx.x % a.parts, row = row0 + blockIdx.x / a.parts;
    const char* base = (const char*)a.logits + row * a.ld * (BF16 ? 2 : 4);
    const int head = min((int)((16 - ((uintptr_t)base & 15)) & 15) / (BF16 ? 2 : 4), a.vocab);
    const int pieces = (a.vocab - head) / V, tiles = (pieces + 64 * kLoads - 1) / (64 * kLoads);
    const int t0 = (int)((long long)tiles * part / a.parts), t1 = (int)((long long)tiles * (part + 1) / a.parts);
    const char* body = base + head * (BF16 ? 2 : 4);
    const uint32_t none = BF16 ? 0xff80ff80u : 0xff800000u;
    u32x4 buf[kLoads];
    const auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int p = (t * kLoads + i) * 64 + lane;
            buf[i] = u32x4{none, none, none, none};
            if (p < pieces) buf[i] = *(const u32x4*)(body + (size_t)p * 16);
        }
    };
    const auto at = [&](int i) {
        return BF16 ? __uint_as_float((uint32_t)((const uint16_t*)base)[i] << 16) : ((const float*)base)[i];
    };
    int target = a.targets ? a.targets[row] : -1;
    if (t0 + wv < t1) fetch(t0 + wv);
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
    Best best = {lists[TOP ? wv : 0], sorts[TOP ? wv : 0], -INFINITY, false, 0, a.top};
    // elements in front (the first step) and behind
    const bool edges = part == 0 && wv == 0;
    const auto single = [&](int id, bool on) {
        const float x = on ? at(id) : -INFINITY;
        const float top = wave_max(x);
        if (top > u.m) raise(u, top, c);
        const float z = on ? (x - (u.m == -INFINITY ? 0.f : u.m)) * c : -INFINITY, w = __builtin_amdgcn_exp2f(z);
        u.s += w;
        u.a += w * __builtin_elementwise_maximum(z, -200.f);
        above += __popcll(__ballot(on && before(x, id, xt, target)));
        if (TOP) push(best, x, id, on);
    };
    if (edges && head) single(lane, lane < head);
    if (edges && tp >= 0 && tp < pieces) {
        const int id = head + tp * V + lane;
        above += __popcll(__ballot(id < target && at(min(id, target)) == xt));
    }
    bool first = true;
    for (int t = t0 + wv; t < t1; t += 4) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = element<BF16>(buf, i);
        if (t + 4 < t1) fetch(t + 4);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < E; ++i) top = fmaxf(top, x[i]);
        if (__any(top > u.m)) raise(u, wave_max(fmaxf(top, u.m)), c);
        const float m = u.m == -INFINITY ? 0.f : u.m;
        float as = 0.f;
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float z = (x[i] - m) * c, w = __builtin_amdgcn_exp2f(z);
            ss += w;
            as = __builtin_fmaf(w, __builtin_elementwise_maximum(z, -200.f), as);
        }
        u.s += ss;
        u.a += as;
        const int id0 = head + (t * kLoads * 64 + lane) * V;
        if (a.targets) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const float reach = (t * kLoads + i) * 64 + lane < tp ? xt : over;
#pragma unroll
                for (int k = 0; k < V; ++k) n += __popcll(__ballot(x[i * V + k] >= reach));
            }
            above += n;
        }
        if (TOP) {
            if (first) best.floor = fmaxf(best.floor, floor_of(top, a.top));
            first = false;
            if (__any(gets_in(best, top))) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    if (best.count > kTight) tighten(best);
                    const bool on = (t * kLoads + i) * 64 + lane < pieces;
#pragma unroll
                    for (int k = 0; k < V; ++k) push(best, x[i * V + k], id0 + i * 64 * V + k, on);
                }
                if (best.count > kTight) tighten(best);
            }
        }
    }
    const int tail = head + pieces * V;
    if (edges && tail < a.vocab) {
        single(tail + lane, tail + lane < a.vocab);
        if (TOP && best.count > kTight) tighten(best);
    }
    u.s = wave_sum_d(u.s);
    u.a = wave_sum_d(u.a);
    if (lane == 0) {
        waves[wv] = {u.s, u.a, u.m, above};
        counts[wv] = best.count;
    }
    __syncthreads();
    const size_t room = blockIdx.x;
    LpPart* parts = (LpPart*)a.ws;
    float2* tops = (float2*)(a.ws + kPartRooms * sizeof(LpPart)) + room * kTopMost;
    if (tid == 0) {
        LpPart p = waves[0];
        for (int w = 1; w < 4; ++w) p.m = fmaxf(p.m, waves[w].m);
        p.s = p.a = 0.0;
        p.above = 0;
        for (int w = 0; w < 4; ++w) {
            const LpPart& q = waves[w];
            p.above += q.above;
            if (q.m == -INFINITY && q.s == 0.0) continue;
            const double z = q.m == p.m ? 0.0 : ((double)q.m - p.m) * a.c, f = exp2(z);
            p.s += f * q.s;
            p.a += f > 0.0 ? f * (q.a + z * q.s) : 0.0;
        }
        parts[room] = p;
    }
    if (TOP) {
        const bool on = lane < counts[wv];
        const float2 mine = on ? lists[wv][lane] : make_float2(-INFINITY, 0.f);
        int r = 0;
        for (int w = 0; w < 4; ++w)
            for (int k = 0; k < counts[w]; ++k) {
                const float2 o = lists[w][k];
                r += before(o.x, __float_as_int(o.y), mine.x, __float_as_int(mine.y));
            }
        if (on && r < a.top) tops[r] = mine;
        int all = 0;
        for (int w = 0; w < 4; ++w) all += counts[w];
        if (tid >= all && tid < a.top) tops[tid] = make_float2(-INFINITY, __int_as_float(0x7fffffff));
    }
}

// Joins a row's parts: a block a row.
template <bool TOP>
__global__ void __launch_bounds__(256) logprobs_join(LogprobArgs a, int row0) {
    __shared__ float2 c[TOP ? kParts * kTopMost : 1];
    __shared__ int kept;
    __shared__ double lse;
    __shared__ float mx;
    const int tid = threadIdx.x, row = row0 + blockIdx.x;
    const LpPart* parts = (const LpPart*)a.ws + (size_t)blockIdx.x * a.parts;
    const float2* tops = (const float2*)(a.ws + kPartRooms * sizeof(LpPart)) + (size_t)blockIdx.x * a.parts * kTopMost;
    if (tid < 64) {
        LpPart p = tid < a.parts ? parts[tid] : LpPart{0.0, 0.0, -INFINITY, 0};
        const float m = wave_max(p.m);
        double s = 0.0, e = 0.0;
        if (tid < a.parts && !(p.m == -INFINITY && p.s == 0.0)) {
            const double z = p.m == m ? 0.0 : ((double)p.m - m) * a.c, f = exp2(z);
            s = f * p.s;
            e = f > 0.0 ? f * (p.a + z * p.s) : 0.0;
        }
        s = wave_sum_d(s);
        e = wave_sum_d(e);
        int above = p.above;
        for (int k = 32; k; k >>= 1) above += __shfl_xor(above, k);
        if (tid == 0) {
            const bool bad = !(s > 0.0) || !(s < INFINITY) || !(m < INFINITY);
            const double l = bad ? (double)NAN : log2(s);
            lse = l;
            mx = m;
            kept = 0;
            const int t = a.targets ? a.targets[row] : -1;
            const bool on = !bad && t >= 0 && t < a.vocab;
            if (a.logprobs) {
                double v = NAN;
                if (on) {
                    const long long i = row * a.ld + t;
                    const float x = a.bf16 ? bf2f(((const uint16_t*)a.logits)[i]) : ((const float*)a.logits)[i];
                    v = (((double)x - m) * a.c - l) * 0.69314718055994530942;
                }
                a.logprobs[row] = (float)v;
            }
            if (a.ranks) a.ranks[row] = on ? above : -1;
            if (a.entropy) a.entropy[row] = (float)((l - e / s) * 0.69314718055994530942);
        }
    }
    if (!TOP) return;
    const int n = a.parts * a.top;
    for (int i = tid; i < n; i += 256) c[i] = tops[i / a.top * kTopMost + i % a.top];
    __syncthreads();
    const long long o = (long long)row * a.top;
    if (!(lse == lse)) {
        if (tid < a.top) {
            if (a.top_ids) a.top_ids[o + tid] = -1;
            if (a.top_logprobs) a.top_logprobs[o + tid] = NAN;
        }
        return;
    }
    for (int i = tid; i < n; i += 256) {
        const float2 mine = c[i];
        int r = 0;
        for (int k = 0; k < n; ++k) r += before(c[k].x, __float_as_int(c[k].y), mine.x, __float_as_int(mine.y));
        if (r < a.top && __float_as_int(mine.y) < a.vocab) {
            if (a.top_ids) a.top_ids[o + r] = __float_as_int(mine.y);
            if (a.top_logprobs)
                a.top_logprobs[o + r] = (float)((((double)mine.x - mx) * a.c - lse) * 0.69314718055994530942);
        }
    }
}

hipError_t launch_logprobs(LogprobArgs a, hipStream_t st) {
    const int el = a.bf16 ? 8 : 4, tiles = (a.vocab / el + 64 * kLoads - 1) / (64 * kLoads);
    a.parts = std::max(1, std::min({kParts, (tiles + 3) / 4, (2048 + a.rows - 1) / a.rows}));
    const int most = kPartRooms / a.parts;
    for (int r = 0, m; r < a.rows; r += m) {
        m = std::min(most, a.rows - r);
        const dim3 grid((unsigned)(m * a.parts));
        const auto k = a.bf16 ? (a.top ? logprobs_kernel<true, true> : logprobs_kernel<true, false>)
                              : (a.top ? logprobs_kernel<false, true> : logprobs_kernel<false, false>);
        hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a, r);
        hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(a.top ? logprobs_join<true> : logprobs_join<false>, dim3(m), dim3(256), 0, st, a, r);
        rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

}  // namespace q35
