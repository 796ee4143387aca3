// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// A lane has k drafts d_0 .. d_{k-1}, k + 1 rows of target logits (row j before draft j, row k after
// the last) and, unless its drafter is certain of its drafts, k rows of the drafter's logits. With
// p_j = softmax(l_j / T) and q_j = softmax(l'_j / T) (1 at the draft for a certain drafter):
//   draft j stays while u_j q_j(d_j) < p_j(d_j); the first that does not ends the lane at row a = j,
//   and its token comes from the weights max(p_a - q_a, 0); without one, from p_a, a = the drafts' number;
//   the token is the first whose running sum of weights exceeds u_k times their total.
// Every token then has the target's distribution, whatever the drafter.
//
// The token is a border between two sums of up to 10^6 terms, so everything here is float64: with
// float32's exp and sums one token in forty at a 248,320-word vocabulary would be another one. The
// logits are read once (verify_stats), and a float64 power of its own (add_power, 11 float64 operations) takes less than a
// logit's load; what follows touches one row of a lane again, or two.
#include "q35_common.h"
#include "q35_kv4.h"

namespace q35 {

// e^((l - m) / T) = 2^(d c), d = l - m <= 0, c = log2(e) / T. d c + 1.5 * 2^52 rounds to a whole number whose low
// bits are the exponent; what is left, |f| <= 1/2, is d c minus it, in one rounding; 2^f is the
// polynomial that interpolates it at the ten Chebyshev points (relative error under 2e-14, far under what
// a border between a million terms notices). 0 under 2^-1074, so also for l = -inf.
typedef VerifyScale Scale;
__device__ __forceinline__ double power(double d, const Scale& sc) {
    d = fmax(d, sc.low);
    const double t = __builtin_fma(d, sc.c, 6755399441055744.0), k = t - 6755399441055744.0;
    const double f = __builtin_fma(d, sc.c, -k);
    double p = 1.0205907319260632e-07;
    p = __builtin_fma(p, f, 1.3259645343488558e-06);
    p = __builtin_fma(p, f, 1.5252672910770481e-05);
    p = __builtin_fma(p, f, 0.00015403433750730278);
    p = __builtin_fma(p, f, 0.0013333558200829426);
    p = __builtin_fma(p, f, 0.009618129193935192);
    p = __builtin_fma(p, f, 0.05550410866465135);
    p = __builtin_fma(p, f, 0.24022650695640335);
    p = __builtin_fma(p, f, 0.6931471805599462);
    p = __builtin_fma(p, f, 1.0000000000000135);
    return __builtin_ldexp(p, (int)(uint32_t)__builtin_bit_cast(unsigned long long, t));
}

// The same added to s, for sums whose largest term is 1: t[i] = 2^(i / 64) (LDS), and 2^f for the rest, |f| <= 1/128, by
// a fourth degree (interpolated likewise; under 5e-15). Exponents end at -990, so the power goes into the bits.
__device__ __forceinline__ void add_power(double& s, double d, const Scale& sc, double low, const double* t) {
    d = fmax(d, low);
    const double w = __builtin_fma(d, sc.c, 105553116266496.0), k = w - 105553116266496.0;   // whole 64ths
    const double f = __builtin_fma(d, sc.c, -k);
    const int n = (int)(uint32_t)__builtin_bit_cast(unsigned long long, w);
    unsigned long long b = __builtin_bit_cast(unsigned long long, t[n & 63]);
    b += (unsigned long long)(((uint32_t)n & ~63u) << 14) << 32;
    double p = 0.009618140859595685;
    p = __builtin_fma(p, f, 0.05550421039186821);
    p = __builtin_fma(p, f, 0.2402265069589214);
    p = __builtin_fma(p, f, 0.6931471805583931);
    p = __builtin_fma(p, f, 1.0);
    s = __builtin_fma(__builtin_bit_cast(double, b), p, s);
}

constexpr int kMaxChunk = 8192;
struct Stat { double m, s; };        // a chunk's largest logit, and the sum of 2^((l - m) c); greedy: its index

// Reductions and running sums over a wave by DPP moves (a shuffle of a double is two trips to LDS, and the last
// kernel is a chain of them): within rows of 16 by 1, 2, 4 and 8 lanes, then row 0 into 1 and 2 into 3, then
// the lower half into the upper. Lane 63 ends with all lanes' result.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or(double v, double none) {
    const unsigned long long w = __builtin_bit_cast(unsigned long long, v), n = __builtin_bit_cast(unsigned long long, none);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)n, (int)(uint32_t)w, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(n >> 32), (int)(uint32_t)(w >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or(int v, int none) { return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false); }
template <class T, class F>
__device__ __forceinline__ T wave_scan(T v, T none, F f) {
    v = f(v, dpp_or<0x111, 0xf>(v, none));       // row_shr:1
    v = f(v, dpp_or<0x112, 0xf>(v, none));
    v = f(v, dpp_or<0x114, 0xf>(v, none));
    v = f(v, dpp_or<0x118, 0xf>(v, none));
    v = f(v, dpp_or<0x142, 0xa>(v, none));       // row_bcast:15
    return f(v, dpp_or<0x143, 0xc>(v, none));    // row_bcast:31
}
__device__ __forceinline__ double last_lane(double v) {
    const unsigned long long w = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)w, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(w >> 32), 63);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double running(double v) { return wave_scan(v, 0.0, [](double x, double y) { return x + y; }); }
__device__ __forceinline__ double wsum(double v) { return last_lane(running(v)); }
__device__ __forceinline__ double wmax(double v) {
    return last_lane(wave_scan(v, -(double)INFINITY, [](double x, double y) { return fmax(x, y); }));
}
__device__ __forceinline__ int wmin_i(int v) {
    return __builtin_amdgcn_readlane(wave_scan(v, 0x7fffffff, [](int x, int y) { return min(x, y); }), 63);
}
__device__ __forceinline__ int wmax_i(int v) {
    return __builtin_amdgcn_readlane(wave_scan(v, -0x7fffffff, [](int x, int y) { return max(x, y); }), 63);
}

// Four (f32) or eight (bf16) logits from i on. Rows may start at any element.
template <bool BF16>
__device__ __forceinline__ void load_whole(const void* row, int i, float* v) {
    uint32_t w[4];
    __builtin_memcpy(w, (const char*)row + (size_t)i * (BF16 ? 2 : 4), 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (BF16) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            v[j] = __uint_as_float(w[j]);
        }
    }
}
// The same with -inf past the vocabulary.
template <bool BF16>
__device__ __forceinline__ void load_logits(const void* row, int i, int vocab, float* v) {
    constexpr int N = BF16 ? 8 : 4;
    if (i + N <= vocab) return load_whole<BF16>(row, i, v);
#pragma unroll
    for (int j = 0; j < N; ++j)
        v[j] = i + j >= vocab ? -INFINITY : BF16 ? bf2f(((const uint16_t*)row)[i + j]) : ((const float*)row)[i + j];
}
template <bool BF16>
__device__ __forceinline__ float logit(const void* row, int i) {
    return BF16 ? bf2f(((const uint16_t*)row)[i]) : ((const float*)row)[i];
}

// Target row j of a lane (j <= k), or draft row j - k - 1, and the place of its stats.
template <bool BF16>
__device__ __forceinline__ const void* row_of(const VerifyArgs& a, int lane, int j) {
    const char* p = j <= a.k ? (const char*)a.logits : (const char*)a.draft_logits;
    const long long r = j <= a.k ? ((long long)lane * (a.k + 1) + j) * a.ld : ((long long)lane * a.k + j - a.k - 1) * a.ldd;
    return p + r * (BF16 ? 2 : 4);
}
__device__ __forceinline__ int rows_of(const VerifyArgs& a) { return a.draft_logits ? 2 * a.k + 1 : a.k + 1; }
__device__ __forceinline__ Stat* stats_of(const VerifyArgs& a, int lane, int j) {
    return (Stat*)a.stats + ((size_t)lane * rows_of(a) + j) * a.chunks;
}

// A block per (chunk, row): the chunk in registers, its maximum, then its sum of exponentials. Bound by HBM: 256 lanes
// x 3 rows of 248,320 float32 logits (763 MB) 132 us, 5.8 TB/s, launched back to back (with waits between 142 to 154, and
// so measured: with a ninth degree in place of the table 174, chunks of 4096 instead of 8192 in turn 158 to 142).
template <bool BF16, int LOADS>
__global__ void __launch_bounds__(256) verify_stats(VerifyArgs a) {
    constexpr int N = BF16 ? 8 : 4;
    __shared__ float mx[4];
    __shared__ double sm[4];
    __shared__ int at[4];
    __shared__ double t[64];
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int c = blockIdx.x % a.chunks, rr = blockIdx.x / a.chunks, j = rr % rows_of(a), ln = rr / rows_of(a);
    const void* row = row_of<BF16>(a, ln, j);
    const int i0 = c * a.chunk;
    float v[LOADS][N];
#pragma unroll
    for (int b = 0; b < LOADS; ++b) {        // (a chunk within the vocabulary: no check a load)
        const int i = i0 + (b * 256 + (int)threadIdx.x) * N;
        if (i0 + a.chunk <= a.vocab) load_whole<BF16>(row, i, v[b]);
        else load_logits<BF16>(row, i, a.vocab, v[b]);
    }
    if (threadIdx.x < 64) t[threadIdx.x] = exp2(threadIdx.x * (1.0 / 64));
    float m = -INFINITY;                 // (a NaN anywhere makes it one)
#pragma unroll
    for (int b = 0; b < LOADS; ++b)
#pragma unroll
        for (int e = 0; e < N; ++e) m = __builtin_elementwise_maximum(m, v[b][e]);
    const bool nan = __any(m != m);
    m = nan ? __uint_as_float(0x7fc00000u) : wave_max(m);
    if (lane == 0) mx[wv] = m;
    __syncthreads();
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx[0], mx[1]), __builtin_elementwise_maximum(mx[2], mx[3]));
    Stat* out = stats_of(a, ln, j) + c;
    if (a.inv_temp == 0.0) {             // greedy: the lowest index of the maximum
        int best = 0x7fffffff;
#pragma unroll
        for (int b = LOADS - 1; b >= 0; --b)
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
                if (v[b][e] == m) best = i0 + (b * 256 + (int)threadIdx.x) * N + e;
        best = wmin_i(best);
        if (lane == 0) at[wv] = best;
        __syncthreads();
        if (threadIdx.x == 0) *out = {(double)m, (double)min(min(at[0], at[1]), min(at[2], at[3]))};
        return;
    }
    double s = 0.0;
    if (m > -INFINITY && m < INFINITY) {
        const Scale sc = a.scale;
        const double md = m, low = sc.low * 0.9;
#pragma unroll
        for (int b = 0; b < LOADS; ++b)
#pragma unroll
            for (int e = 0; e < N; ++e) add_power(s, (double)v[b][e] - md, sc, low, t);
    }
    s = wsum(s);
    if (lane == 0) sm[wv] = s;
    __syncthreads();
    if (threadIdx.x == 0) *out = {(double)m, (sm[0] + sm[1]) + (sm[2] + sm[3])};
}

// A row's maximum and sum from its chunks' (chunk i * 64 + lane in v[i]), by one wave; greedy: the maximum
// and its lowest index.
constexpr int kMaxChunks = 512;
template <int N>
__device__ __forceinline__ void load_stats(const VerifyArgs& a, const Stat* st, Stat* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = i * 64 + (threadIdx.x & 63);
        v[i] = {-INFINITY, 0.0};
        if (c < a.chunks) v[i] = st[c];
    }
}
template <int N>
__device__ __forceinline__ Stat row_stat(const VerifyArgs& a, const Stat* v, const Scale& sc) {
    double m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) { m = fmax(m, v[i].m); nan |= v[i].m != v[i].m; }
    m = wmax(m);
    if (__any(nan)) m = __longlong_as_double(0x7ff8000000000000ll);
    double s = 0.0;
    if (a.inv_temp == 0.0) {
        s = 2147483647.0;
#pragma unroll
        for (int i = 0; i < N; ++i) if (v[i].m == m) s = fmin(s, v[i].s);
        s = -wmax(-s);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) if (v[i].s > 0.0) s += v[i].s * power(v[i].m - m, sc);
        s = wsum(s);
    }
    return {m, s};
}
// A row with a NaN, an infinity above or nothing but -inf has no distribution.
__device__ __forceinline__ bool has_dist(const Stat& s) { return s.m > -INFINITY && s.m < INFINITY; }

// What becomes of a lane: its accepted drafts, and where its token comes from.
enum { kFromTarget = 0, kNotDraft = 1, kRest = 2, kNoToken = 3, kArgmax = 4 };
struct Fate {
    int accepted, kind, draft;
    Stat p, q;                       // of target row `accepted`; of its draft row (kRest)
};

// All waves make the lane's row statistics into rs (row order of row_of), k threads the drafts' probabilities
// into pq; then every thread decides alike.
struct Draft { int id; double p, q; };
template <bool BF16, int WAVES>
__device__ __forceinline__ Fate decide_kind(const VerifyArgs& a, int ln, const Scale& sc, Stat* rs, Draft* pq) {
    const int wv = threadIdx.x >> 6, tid = threadIdx.x;
    const bool greedy = a.inv_temp == 0.0;
    Draft d = {-1, 0.0, 1.0};
    float lp = -INFINITY, lq = -INFINITY;
    if (tid < a.k) {
        d.id = a.drafts[(size_t)ln * a.k + tid];
        if (d.id >= 0 && d.id < a.vocab && !greedy) {
            lp = logit<BF16>(row_of<BF16>(a, ln, tid), d.id);
            if (a.draft_logits) lq = logit<BF16>(row_of<BF16>(a, ln, a.k + 1 + tid), d.id);
        }
    }
    if (a.chunks <= 64) {                    // a wave's rows in flight together
        constexpr int kMine = (2 * kVerifyDrafts + 1 + WAVES - 1) / WAVES;
        Stat v[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (wv + i * WAVES < rows_of(a)) load_stats<1>(a, stats_of(a, ln, wv + i * WAVES), v + i);
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (wv + i * WAVES < rows_of(a)) {
                const Stat s = row_stat<1>(a, v + i, sc);
                if ((tid & 63) == 0) rs[wv + i * WAVES] = s;
            }
    } else {
        for (int j = wv; j < rows_of(a); j += WAVES) {
            Stat v[kMaxChunks / 64];
            load_stats<kMaxChunks / 64>(a, stats_of(a, ln, j), v);
            const Stat s = row_stat<kMaxChunks / 64>(a, v, sc);
            if ((tid & 63) == 0) rs[j] = s;
        }
    }
    __syncthreads();
    if (tid < a.k) {
        const Stat ps = rs[tid];
        d.p = has_dist(ps) ? power((double)lp - ps.m, sc) / ps.s : 0.0;
        if (a.draft_logits) {
            const Stat qs = rs[a.k + 1 + tid];
            d.q = has_dist(qs) ? power((double)lq - qs.m, sc) / qs.s : 0.0;
        }
        pq[tid] = d;
    }
    __syncthreads();
    const float* u = a.u + (size_t)ln * (a.k + 1);
    for (int j = 0; j < a.k; ++j) {
        const int t = pq[j].id;
        const bool dist = has_dist(rs[j]);
        if (t < 0) return {j, !dist ? kNoToken : greedy ? kArgmax : kFromTarget, -1, {}, {}};
        if (greedy) {
            if (dist && (double)t == rs[j].s) continue;
            return {j, dist ? kArgmax : kNoToken, t, {}, {}};
        }
        const bool qd = !a.draft_logits || has_dist(rs[a.k + 1 + j]);
        if (qd && (double)u[j] * pq[j].q < pq[j].p) continue;
        const int from = a.draft_logits ? kRest : kNotDraft;
        return {j, !dist ? kNoToken : qd && (a.draft_logits || t < a.vocab) ? from : kFromTarget, t, {}, {}};
    }
    return {a.k, !has_dist(rs[a.k]) ? kNoToken : greedy ? kArgmax : kFromTarget, -1, {}, {}};
}
template <bool BF16, int WAVES>
__device__ __forceinline__ Fate decide(const VerifyArgs& a, int ln, const Scale& sc, Stat* rs, Draft* pq) {
    Fate f = decide_kind<BF16, WAVES>(a, ln, sc, rs, pq);
    f.p = rs[f.accepted];
    if (f.kind == kRest) f.q = rs[a.k + 1 + f.accepted];
    return f;
}

// The weight of token i of the lane's row: p up to a factor, without the draft, or max(p - q, 0).
template <bool BF16>
struct Weights {
    const void *pr, *qr;
    Scale sc;
    double pm, qm, pz, qz;           // maxima, 1 / sums (kRest)
    int kind, draft, vocab;
    __device__ __forceinline__ Weights(const VerifyArgs& a, int ln, const Fate& ft, const Scale& sc_)
        : sc(sc_), kind(ft.kind), draft(ft.draft), vocab(a.vocab) {
        pr = row_of<BF16>(a, ln, ft.accepted);
        pm = ft.p.m;
        pz = 1.0 / ft.p.s;
        if (kind == kRest) {
            qr = row_of<BF16>(a, ln, a.k + 1 + ft.accepted);
            qm = ft.q.m;
            qz = 1.0 / ft.q.s;
        }
    }
    // of N tokens from i on; 0 past the vocabulary
    template <int N>
    __device__ __forceinline__ void at(int i, double* w) const {
        constexpr int L = BF16 ? 8 : 4;
        float v[N];
#pragma unroll
        for (int b = 0; b < N; b += L) load_logits<BF16>(pr, i + b, vocab, v + b);
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = power((double)v[e] - pm, sc);
        if (kind == kRest) {
#pragma unroll
            for (int b = 0; b < N; b += L) load_logits<BF16>(qr, i + b, vocab, v + b);
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = fmax(w[e] * pz - power((double)v[e] - qm, sc) * qz, 0.0);
        } else if (kind == kNotDraft) {
#pragma unroll
            for (int e = 0; e < N; ++e) if (i + e == draft) w[e] = 0.0;
        }
    }
};

// With a drafter's probabilities: the lanes' decisions, kept for verify_token, and the chunks' sums of max(p - q, 0)
// for those that draw from it. A block per (chunk, lane); each block decides for itself, which costs less than another
// launch would. 17 lanes x 4 drafts of 32,003 bfloat16 logits: 7.4 us, most of it the chain from the drafts to the
// decision to the row.
template <bool BF16>
__global__ void __launch_bounds__(256) verify_rest(VerifyArgs a, double* rest, Fate* fates) {
    __shared__ Stat rs[2 * kVerifyDrafts + 1];
    __shared__ Draft pq[kVerifyDrafts];
    __shared__ double sm[4];
    const int c = blockIdx.x % a.chunks, ln = blockIdx.x / a.chunks;
    const Scale sc = a.scale;
    const Fate ft = decide<BF16, 4>(a, ln, sc, rs, pq);
    if (c == 0 && threadIdx.x == 0) fates[ln] = ft;
    if (ft.kind != kRest) return;
    const Weights<BF16> wt(a, ln, ft, sc);
    double s = 0.0;
    for (int i = c * a.chunk + (int)threadIdx.x * 8; i < min((c + 1) * a.chunk, a.vocab); i += 2048) {
        double w[8];
        wt.template at<8>(i, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += w[e];
    }
    s = wsum(s);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) rest[(size_t)ln * a.chunks + c] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// Inclusive sum over the block's 1024 threads, by place; part: 16 doubles.
__device__ __forceinline__ double block_scan(double v, double* part) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    v = running(v);
    __syncthreads();
    if (lane == 63) part[wv] = v;
    __syncthreads();
    double before = 0.0;
#pragma unroll
    for (int w = 0; w < 15; ++w) before += w < wv ? part[w] : 0.0;
    return before + v;
}
// The lowest `first` and the highest `last` of the block's threads.
__device__ __forceinline__ int2 block_ends(int first, int last, int2* ends) {
    first = wmin_i(first);
    last = wmax_i(last);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) ends[threadIdx.x >> 6] = make_int2(first, last);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) { first = min(first, ends[w].x); last = max(last, ends[w].y); }
    return make_int2(first, last);
}

// A block per lane: the decision, the chunk that holds the border, the token in it. One lane 7.0 us, 256 lanes 12.9: a
// chain of four trips to memory and five block-wide sums. (Joined to verify_stats by its last blocks it would need a
// device-wide release a block, which writes the caches back: 1256 us instead of 164 + 15; by relaxed counts 283.)
template <bool BF16>
__global__ void __launch_bounds__(1024) verify_token(VerifyArgs a, const double* rest, const Fate* fates) {
    __shared__ Stat rs[2 * kVerifyDrafts + 1];
    __shared__ Draft pq[kVerifyDrafts];
    __shared__ double part[16], total, base;
    __shared__ int2 ends[16];
    const int ln = blockIdx.x, tid = threadIdx.x;
    const Scale sc = a.scale;
    const Fate ft = a.draft_logits ? fates[ln] : decide<BF16, 16>(a, ln, sc, rs, pq);
    int token = -1;
    if (ft.kind == kArgmax) token = (int)ft.p.s;
    if (ft.kind < kNoToken) {
        Weights<BF16> wt(a, ln, ft, sc);
        int pick = -1;
        double border = 0.0;
        for (int pass = 0; pass < 2 && pick < 0; ++pass) {
            double cw = 0.0;                 // this thread's chunk
            if (tid < a.chunks) {
                const Stat st = stats_of(a, ln, ft.accepted)[tid];
                cw = wt.kind == kRest ? rest[(size_t)ln * a.chunks + tid]
                     : st.s > 0.0 ? st.s * power(st.m - wt.pm, sc) : 0.0;
            }
            if (wt.kind == kNotDraft) {      // the draft's chunk, summed without it
                const int c = ft.draft / a.chunk;
                double w[8], s = 0.0;
                if (tid * 8 < a.chunk) {
                    wt.template at<8>(c * a.chunk + tid * 8, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s += w[e];
                }
                s = block_scan(s, part);
                if (tid == 1023) total = s;
                __syncthreads();
                if (tid == c) cw = total;
                __syncthreads();
            }
            const double run = block_scan(cw, part);
            if (tid == 1023) total = run;
            __syncthreads();
            border = (double)a.u[(size_t)ln * (a.k + 1) + a.k] * total;
            const int2 at = block_ends(cw > 0.0 && run > border ? tid : 0x7fffffff, cw > 0.0 ? tid : -1, ends);
            pick = at.x < a.chunks ? at.x : at.y;
            if (tid == pick) base = run - cw;
            wt.kind = pick < 0 ? (int)kFromTarget : wt.kind;   // nothing is left of p - q (or of p without the draft): p itself
        }
        if (pick >= 0) {
            const int i = pick * a.chunk + tid * 8;
            double w[8], mine = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 0.0;
            if (tid * 8 < a.chunk) wt.template at<8>(i, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) mine += w[e];
            double run = block_scan(mine, part);
            run = base + (run - mine);
            int first = 0x7fffffff, last = -1;       // the first past the border, and the last with any weight
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                run += w[e];
                if (w[e] > 0.0) {
                    last = i + e;
                    if (run > border && first == 0x7fffffff) first = i + e;
                }
            }
            const int2 at = block_ends(first, last, ends);
            token = at.x < a.vocab ? at.x : at.y;
        }
    }
    if (tid == 0) a.accepted[ln] = ft.accepted;
    if (tid <= a.k) a.tokens[(size_t)ln * (a.k + 1) + tid] = tid < ft.accepted ? a.drafts[(size_t)ln * a.k + tid] : tid == ft.accepted ? token : -1;
}

// Chunks of 8192 logits, fewer while the rows are too few to fill the card with them (2048 is the
// least); vocab <= 2^20 keeps a row at kMaxChunks or less.
static int chunk_of(long long rows, int vocab) {
    int chunk = kMaxChunk;
    while (chunk > 2048 && rows * ((vocab + chunk - 1) / chunk) < 1024) chunk /= 2;
    return chunk;
}
size_t verify_ws_doubles(int max_rows) {
    // (chunk sums of the rows, of the lanes, the lanes' decisions)
    // 2 max_rows rows of up to 128 chunks of 8192, or fewer rows of smaller chunks: under 1024 chunks
    // at twice their size, so at most 2048 and one more a row
    const size_t rows = 2 * (size_t)max_rows;
    return 2 * (rows * 128 + 2048 + rows) + (rows * 128 + 2048 + rows) + sizeof(Fate) / 8 * (size_t)max_rows;
}

template <bool BF16>
static hipError_t launch_v(VerifyArgs& a, hipStream_t st) {
    const int per = a.draft_logits ? 2 * a.k + 1 : a.k + 1;
    a.chunk = chunk_of((long long)a.n * per, a.vocab);
    a.chunks = (a.vocab + a.chunk - 1) / a.chunk;
    double* rest = a.stats + 2 * (size_t)a.n * per * a.chunks;
    Fate* fates = (Fate*)(rest + (size_t)a.n * a.chunks);
    const dim3 grid((unsigned)a.chunks * a.n * per);
    constexpr int N = BF16 ? 8 : 4;
    if (a.chunk == 8192) hipLaunchKernelGGL((verify_stats<BF16, 32 / N>), grid, dim3(256), 0, st, a);
    else if (a.chunk == 4096) hipLaunchKernelGGL((verify_stats<BF16, 16 / N>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((verify_stats<BF16, 8 / N>), grid, dim3(256), 0, st, a);
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    if (a.draft_logits && a.inv_temp != 0.0) {
        hipLaunchKernelGGL(verify_rest<BF16>, dim3((unsigned)a.chunks * a.n), dim3(256), 0, st, a, rest, fates);
        if ((rc = hipGetLastError()) != hipSuccess) return rc;
    }
    hipLaunchKernelGGL(verify_token<BF16>, dim3(a.n), dim3(1024), 0, st, a, (const double*)rest, (const Fate*)fates);
    return hipGetLastError();
}
hipError_t launch_verify(VerifyArgs& a, hipStream_t st) { return a.bf16 ? launch_v<true>(a, st) : launch_v<false>(a, st); }

}  // namespace q35
