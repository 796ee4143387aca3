// Head norms with rotation, the 4-bit K/V cache, and the attention that reads it.
#include <algorithm>
#include <cstring>

#include "q35_common.h"
#include "q35_kv4.h"

namespace q35 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The pair of values in byte SEL of w, times the power of two in `scale`'s exponent: exact; NaN
// where that exponent is 255 (all 256 bytes x 245 scales and 255 compared on MI355X).
template <int SEL>
__device__ __forceinline__ uint32_t two_values(uint32_t w, float scale) {
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// ------------------------------------------------------------------ norms, rotation, append
// sin and cos of a quarter turn's worth around 0 by their Taylor series in float64 (|r| <= pi / 4:
// the first terms left out are below 2^-54).
__device__ __forceinline__ void sincos_small(double r, double& s, double& c) {
    const double z = r * r;
    double a = 1.0 / 355687428096000.0, b = 1.0 / 20922789888000.0;
    a = __builtin_fma(a, z, -1.0 / 1307674368000.0);
    b = __builtin_fma(b, z, -1.0 / 87178291200.0);
    a = __builtin_fma(a, z, 1.0 / 6227020800.0);
    b = __builtin_fma(b, z, 1.0 / 479001600.0);
    a = __builtin_fma(a, z, -1.0 / 39916800.0);
    b = __builtin_fma(b, z, -1.0 / 3628800.0);
    a = __builtin_fma(a, z, 1.0 / 362880.0);
    b = __builtin_fma(b, z, 1.0 / 40320.0);
    a = __builtin_fma(a, z, -1.0 / 5040.0);
    b = __builtin_fma(b, z, -1.0 / 720.0);
    a = __builtin_fma(a, z, 1.0 / 120.0);
    b = __builtin_fma(b, z, 1.0 / 24.0);
    a = __builtin_fma(a, z, -1.0 / 6.0);
    b = __builtin_fma(b, z, -0.5);
    s = __builtin_fma(r * z, a, r);
    c = __builtin_fma(z, b, 1.0);
}
// cos and sin of pos * theta^(-2 i / rot). In turns the whole part drops out exactly, so a far
// position keeps its angle: float32 angles are off by up to 4e-3 at position 1e5.
__device__ __forceinline__ float2 turn(int pos, int i, int rot, double log2_theta) {
    constexpr double kInv2Pi = 0.15915494309189533577;
    double u = (double)pos * (exp2(-2.0 * i / rot * log2_theta) * kInv2Pi);
    u -= rint(u);
    const double q = rint(4.0 * u);
    double s, c;
    sincos_small((u - 0.25 * q) * 6.283185307179586477, s, c);
    const int k = (int)q & 3;
    const double cc = k & 1 ? -s : c, ss = k & 1 ? c : s;
    return k & 2 ? make_float2((float)-cc, (float)-ss) : make_float2((float)cc, (float)ss);
}

__device__ __forceinline__ float4 load4(const uint16_t* p) {
    const uint2 w = *(const uint2*)p;
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}

// One wave per row and unit of 256 dims (256 / D heads of q, of k or of v), four dims a lane. What it
// writes is decided by borders (a code's midpoints, a scale's step), so every float32 operation is one
// rounding in the stated order, and the sum of squares, the root and the angles are float64.
template <int D>
__global__ void __launch_bounds__(256) heads_kernel(HeadArgs a, int rows, int units) {
    constexpr int kPer = 256 / D;            // heads of a unit
    constexpr int kLanes = D / 4;            // lanes of a head
    __shared__ float xs[4][256];
    __shared__ float2 cs[4][128];
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + wv;
    const int r = (int)(w / units);
    if (r >= rows) return;                   // whole waves; no block barrier below
    int u = (int)(w % units);
    const int qu = a.q.p ? (a.q_heads + kPer - 1) / kPer : 0, ku = (a.kv_heads + kPer - 1) / kPer;
    const int kind = u < qu ? 0 : u < qu + ku ? 1 : 2;
    u -= kind == 0 ? 0 : kind == 1 ? qu : qu + ku;
    const int heads = kind == 0 ? a.q_heads : a.kv_heads;
    const int h = u * kPer + lane / kLanes, d0 = lane % kLanes * 4;
    const bool on = h < heads;
    const int seq = r / a.T, t = r - seq * a.T, pos = a.pos[seq] + t;
    const HeadView in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const HeadView out = kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) x = load4(in.p + r * in.row + h * in.head + d0);
    if (kind < 2) {
        double ss = ((double)(x.x * x.x) + (double)(x.y * x.y)) + ((double)(x.z * x.z) + (double)(x.w * x.w));
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1) ss += __shfl_xor(ss, o);
        const float rs = (float)(1.0 / sqrt(ss / D + a.eps));
        const float4 nw = load4((kind == 0 ? a.q_norm : a.k_norm) + d0);
        x.x = x.x * rs * (1.0f + nw.x);
        x.y = x.y * rs * (1.0f + nw.y);
        x.z = x.z * rs * (1.0f + nw.z);
        x.w = x.w * rs * (1.0f + nw.w);
        const int half = a.rot / 2;
        for (int i = lane; i < half; i += 64) cs[wv][i] = turn(pos, i, a.rot, a.log2_theta);
        *(float4*)&xs[wv][lane * 4] = x;
        wave_sync();
        const float* hx = &xs[wv][lane / kLanes * D];
        float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = d0 + e;
            if (d < half) {
                const float2 c = cs[wv][d];
                y[e] = y[e] * c.x - hx[d + half] * c.y;
            } else if (d < a.rot) {
                const float2 c = cs[wv][d - half];
                y[e] = y[e] * c.x + hx[d - half] * c.y;
            }
        }
        x = make_float4(y[0], y[1], y[2], y[3]);
    }
    if (kind == 0 || !a.cache) {
        if (on && out.p) {
            uint2 o;
            o.x = f2bf2(x.x, x.y);
            o.y = f2bf2(x.z, x.w);
            *(uint2*)(const_cast<uint16_t*>(out.p) + r * out.row + h * out.head + d0) = o;
        }
        return;
    }
    // the group's largest magnitude as bits (eight lanes): an infinity or a NaN is the largest of all
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint((&x.x)[e]) & 0x7fffffffu);
#pragma unroll
    for (int o = 4; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    // top = 1.m 2^E: 6 * 2^(E - 2) covers it up to m = 0.5, else one step more. Kept within 2^-119 ..
    // 2^125, so that no value of a group overflows bf16 or loses bits below its normal range.
    uint32_t b = max((int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u), 8);
    b = top >= 0x7f800000u ? 255u : min(b, 252u);
    const float sc = scale_of(b);
    uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x.x, x.y, sc, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x.z, x.w, sc, 1);
    if (!on) return;
    if (out.p) {
        uint2 o;
        o.x = two_values<0>(code, sc);
        o.y = two_values<1>(code, sc);
        *(uint2*)(const_cast<uint16_t*>(out.p) + r * out.row + h * out.head + d0) = o;
    }
    uint8_t* tile = a.cache + a.lane[seq] * a.lane_bytes + h * a.region + (size_t)(pos >> 5) * kv4_tile_bytes(D);
    const int tk = pos & 31;
    *(uint16_t*)(tile + (kind == 1 ? kv4_k_code(D, tk, d0) : kv4_v_code(D, tk, d0))) = (uint16_t)code;
    if ((lane & 7) == 0) tile[kind == 1 ? kv4_k_scale(D, tk, d0 >> 5) : kv4_v_scale(D, tk, d0 >> 5)] = (uint8_t)b;
}

hipError_t launch_heads(const HeadArgs& a, int n, hipStream_t st) {
    const int per = 256 / a.D, qu = a.q.p ? (a.q_heads + per - 1) / per : 0, ku = (a.kv_heads + per - 1) / per;
    const int units = qu + ku * (a.v.p ? 2 : 1), rows = n * a.T;
    const long long blocks = ((long long)rows * units + 3) / 4;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    auto k = a.D == 256 ? heads_kernel<256> : a.D == 128 ? heads_kernel<128> : heads_kernel<64>;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, a, rows, units);
    return hipGetLastError();
}

// ------------------------------------------------------------------ rows in and out of the cache
// A thread per 8 dims of a (lane, kv head, slot): 4 bytes of codes, and a scale byte in one of four.
template <bool WRITE>
__global__ void __launch_bounds__(256) kv4_copy_kernel(Kv4Copy a) {
    const int per = a.D / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long rows = (long long)a.n_lanes * a.kv_heads * a.n_slots;
    const long long row = i / per;
    if (row >= rows) return;
    const int d = (int)(i % per) * 8, s = (int)(row % a.n_slots), slot = a.slot0 + s;
    const int lh = (int)(row / a.n_slots);
    uint8_t* tile = a.cache + (size_t)(a.lane0 + lh / a.kv_heads) * a.lane_bytes + lh % a.kv_heads * a.region +
                    (size_t)(slot >> 5) * kv4_tile_bytes(a.D);
    const int tk = slot & 31;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        uint8_t* rowp = (v ? a.vc : a.kc) + row * (a.D / 2) + d / 2;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            uint8_t* c = tile + (v ? kv4_v_code(a.D, tk, d + e) : kv4_k_code(a.D, tk, d + e));
            if (WRITE) *c = rowp[e / 2];
            else rowp[e / 2] = *c;
        }
        if (d % 32 == 0) {
            uint8_t* c = tile + (v ? kv4_v_scale(a.D, tk, d / 32) : kv4_k_scale(a.D, tk, d / 32));
            uint8_t* o = (v ? a.vs : a.ks) + row * (a.D / 32) + d / 32;
            if (WRITE) *c = *o;
            else *o = *c;
        }
    }
}
hipError_t launch_kv4_copy(const Kv4Copy& a, bool write, hipStream_t st) {
    const long long n = (long long)a.n_lanes * a.kv_heads * a.n_slots * (a.D / 8), blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (write) hipLaunchKernelGGL(kv4_copy_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(kv4_copy_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------ attention
// Rows of one sequence and kv head: the T new rows times the head's `group` query heads, row rho =
// t * group + g at position pos + t. S^T = K Q^T and O^T = V^T P^T on 16x16x32 bf16 MFMAs with the
// slots (S^T) and the dims (O^T) in M and 16 rows in N: a lane's column is one row in both, so the row's
// maximum, sum and rescale live in the lane, and S^T's accumulators are P^T's operand as they are.
template <int D>
struct Tile {
    u32x4 k[D / 64], v[D / 64];
    uint32_t ks;
    uint2 vs;
};
template <int D>
__device__ __forceinline__ Tile<D> load_tile(const uint8_t* region, int tile) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const uint8_t* p = region + (size_t)tile * kv4_tile_bytes(D);
    Tile<D> t;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) t.k[i] = __builtin_nontemporal_load((const u32x4*)(p + i * 1024 + lane * 16));
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
        t.v[i] = __builtin_nontemporal_load((const u32x4*)(p + 16 * D + i * 1024 + lane * 16));
    if (D == 256) t.ks = *(const uint32_t*)(p + 32 * D + lane * 4);
    else t.ks = *(const uint16_t*)(p + 32 * D + (D == 64 ? (g >> 1) * 16 + m : lane) * 2);
    t.vs = *(const uint2*)(p + 33 * D + m * D / 512 * 32 + g * 8);
    return t;
}
template <int D>
__device__ __forceinline__ float k_scale(const Tile<D>& t, int half, int s) {
    return scale_of((t.ks >> (D == 256 ? half * 16 + s / 4 * 8 : half * 8)) & 255u);
}
template <int D>
__device__ __forceinline__ q35_bf16x8 k_frag(const Tile<D>& t, int half, int s) {
    const int w = half * (D / 32) + s;
    const uint32_t c = t.k[w / 4][w % 4];
    const float sc = k_scale<D>(t, half, s);
    const u32x4 r = {two_values<0>(c, sc), two_values<1>(c, sc), two_values<2>(c, sc), two_values<3>(c, sc)};
    return __builtin_bit_cast(q35_bf16x8, r);
}
// The dims d and d + 1 (of the lane's D / 16; d even) of its 8 slots as the operands of two MFMAs.
template <int D, int d>
__device__ __forceinline__ void v_frags(const Tile<D>& t, const float* vs, q35_bf16x8& lo, q35_bf16x8& hi) {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int byte = (2 * i + e) * (D / 32) + d / 2;
            const uint32_t c = t.v[byte / 16][byte % 16 / 4];
            const float sc = vs[2 * i + e];
            w[e] = byte % 4 == 0 ? two_values<0>(c, sc) : byte % 4 == 1 ? two_values<1>(c, sc)
                 : byte % 4 == 2 ? two_values<2>(c, sc) : two_values<3>(c, sc);
        }
        a[i] = __builtin_amdgcn_perm(w[1], w[0], 0x05040100u);
        b[i] = __builtin_amdgcn_perm(w[1], w[0], 0x07060302u);
    }
    lo = __builtin_bit_cast(q35_bf16x8, a);
    hi = __builtin_bit_cast(q35_bf16x8, b);
}

// Which slots a row sees: (pos - window, pos] and [0, sinks); window 0: [0, pos].
struct Sight { int pos, low, sinks; };
__device__ __forceinline__ bool sees(const Sight& s, int slot) { return slot <= s.pos && (slot >= s.low || slot < s.sinks); }

// The running state of NQ x 16 rows over the tiles of one wave.
template <int D, int NQ>
struct Rows {
    float m[NQ], l[NQ];          // of row n: its maximum (log2 units), the lane group's share of its sum
    uint32_t bad[NQ];            // groups of 32 dims whose V held a NaN at a slot the row sees
    f32x4 o[NQ][D / 16];         // O^T: dims (4 g + r) D / 16 + i of row n in o[.][i][r]
};

template <int D, int NQ>
__device__ __forceinline__ void tile_step(const Tile<D>& t, const uint8_t* tile_p, int slot0, bool edge,
                                          const q35_bf16x8 (*qf)[D / 32], const Sight* sight, float scale2,
                                          Rows<D, NQ>& st) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    f32x4 s[NQ][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c = 0; c < NQ; ++c) s[c][half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const q35_bf16x8 kf = k_frag<D>(t, half, k);
#pragma unroll
            for (int c = 0; c < NQ; ++c)
                s[c][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[c][k], s[c][half], 0, 0, 0);
        }
    }
#pragma unroll
    for (int c = 0; c < NQ; ++c) { s[c][0] *= scale2; s[c][1] *= scale2; }     // before the mask: scale may be 0 or negative
    uint2 vsb = t.vs;
    // A slot some row may not see: its score is dropped, and a NaN group of V there must not meet the
    // zero weight. Such a group is read as finite and noted for the rows that do see it.
    if (edge) {
        const auto has255 = [](uint32_t w) { return ((~w - 0x01010101u) & w & 0x80808080u) != 0; };
        const bool nan = __any(has255(vsb.x) || has255(vsb.y));
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            uint32_t seen = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool ok = sees(sight[c], slot0 + (j >> 2) * 16 + 4 * g + (j & 3));
                if (!ok) s[c][j >> 2][j & 3] = -INFINITY;
                seen |= (uint32_t)ok << j;
            }
            if (nan)
                for (int b = 0; b < D / 32; ++b) {
                    const uint8_t* p = tile_p + 33 * D + b * 32 + g * 8;
                    for (int j = 0; j < 8; ++j)
                        if (((seen >> j) & 1) && p[j] == 255) st.bad[c] |= 1u << b;
                }
        }
        if (nan) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (((vsb.x >> 8 * j) & 255u) == 255u) vsb.x &= ~(128u << 8 * j);
                if (((vsb.y >> 8 * j) & 255u) == 255u) vsb.y &= ~(128u << 8 * j);
            }
        }
    }
    q35_bf16x8 pf[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, s[c][j >> 2][j & 3]);
        top = fmaxf(top, xor16(top));
        top = fmaxf(top, xor32(top));
        const float mn = fmaxf(st.m[c], top);
        const float ms = mn == -INFINITY ? 0.f : mn;      // nothing seen so far: e^(-inf) stays 0
        if (__any(mn > st.m[c])) {
            const float al = __builtin_amdgcn_exp2f(st.m[c] - ms);
            st.l[c] *= al;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) st.o[c][i] *= al;
            st.m[c] = mn;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = __builtin_amdgcn_exp2f(s[c][j >> 2][j & 3] - ms);
            st.l[c] += p[j];
        }
        // weights of 2^-9 relative rounding for the bf16 product; their sum stays float32
        const u32x4 pw = {f2bf2(p[0], p[1]), f2bf2(p[2], p[3]), f2bf2(p[4], p[5]), f2bf2(p[6], p[7])};
        pf[c] = __builtin_bit_cast(q35_bf16x8, pw);
    }
    float vs[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        vs[j] = scale_of((vsb.x >> 8 * j) & 255u);
        vs[4 + j] = scale_of((vsb.y >> 8 * j) & 255u);
    }
    auto pv = [&](auto dc) {
        constexpr int d = decltype(dc)::value;
        if constexpr (d < D / 16) {
            q35_bf16x8 lo, hi;
            v_frags<D, d>(t, vs, lo, hi);
#pragma unroll
            for (int c = 0; c < NQ; ++c) {
                st.o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, pf[c], st.o[c][d], 0, 0, 0);
                st.o[c][d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, pf[c], st.o[c][d + 1], 0, 0, 0);
            }
        }
    };
    pv(std::integral_constant<int, 0>{});
    pv(std::integral_constant<int, 2>{});
    pv(std::integral_constant<int, 4>{});
    pv(std::integral_constant<int, 6>{});
    pv(std::integral_constant<int, 8>{});
    pv(std::integral_constant<int, 10>{});
    pv(std::integral_constant<int, 12>{});
    pv(std::integral_constant<int, 14>{});
}

// The tiles that rows at positions p0 .. p1 read: those of the sinks, then those from the first row's
// window on. Tile i of the list is i (i < sink) or i - sink + main.
struct TileList { int sink, main, count; };
__host__ __device__ inline TileList tile_list(int p0, int p1, int window, int sinks) {
    const int low = window > 0 && p0 - window + 1 > 0 ? p0 - window + 1 : 0;
    const int sk = sinks < low ? sinks : low;
    TileList t;
    t.main = low >> 5;
    t.sink = (sk + 31) >> 5;
    if (t.sink > t.main) t.sink = t.main;
    t.count = t.sink + (p1 >> 5) - t.main + 1;
    return t;
}

constexpr int kSplitRows = 16;       // rows of one partial result
constexpr int kMaxSplits = 2048;     // partial results of one launch (workspace)
size_t kv4_part_floats() { return (size_t)kMaxSplits * kSplitRows * (256 + 4); }

// Sequence of item z by bisection of first[].
__device__ __forceinline__ int find_seq(const uint16_t* first, int n, int z) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= z) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Decode and verify rows: a block per (sequence, split of its tiles, kv head, NQ x 16 rows), its four
// waves on every fourth tile with the next one's loads in flight, their states joined through LDS.
template <int D, int NQ>
__global__ void __launch_bounds__(256) attn_kv4_kernel(Kv4Attn a, int n, int row_tiles) {
    __shared__ float os[4][16][D + 4];
    __shared__ float ms[4][16], ls[4][16];
    __shared__ uint32_t bs[4][16];
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, nn = lane & 15, g = lane >> 4;
    const int rt = blockIdx.x % row_tiles, h = blockIdx.x / row_tiles % a.kv_heads, z = blockIdx.x / (row_tiles * a.kv_heads);
    const int seq = find_seq(a.first, n, z), split = z - a.first[seq], splits = a.first[seq + 1] - a.first[seq];
    const int group = a.q_heads / a.kv_heads, rows = a.T * group, rho0 = rt * NQ * 16, pos = a.pos[seq];
    const int rho1 = min(rho0 + NQ * 16, rows) - 1;
    const TileList tl = tile_list(pos + rho0 / group, pos + rho1 / group, a.window, a.sinks);
    const int t0 = (int)((long long)tl.count * split / splits), t1 = (int)((long long)tl.count * (split + 1) / splits);
    const uint8_t* region = a.cache + a.lane[seq] * a.lane_bytes + h * a.region;

    q35_bf16x8 qf[NQ][D / 32];
    Sight sight[NQ];
    Rows<D, NQ> st;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int rho = min(rho0 + c * 16 + nn, rows - 1), t = rho / group;
        const uint16_t* q = a.q.p + ((long long)seq * a.T + t) * a.q.row + (h * group + rho - t * group) * a.q.head;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) qf[c][k] = *(const q35_bf16x8*)(q + g * (D / 4) + 8 * k);
        sight[c] = {pos + t, a.window > 0 ? pos + t - a.window + 1 : 0, a.sinks};
        st.m[c] = -INFINITY;
        st.l[c] = 0.f;
        st.bad[c] = 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) st.o[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // tiles whose every slot every row of the block sees: from the last row's window to the first row's slot
    const int full0 = a.window > 0 ? max(pos + rho1 / group - a.window + 1, 0) : 0, full1 = pos + rho0 / group;
    const float scale2 = a.scale * 1.44269504088896f;
    auto at = [&](int i) { return i < tl.sink ? i : i - tl.sink + tl.main; };
    if (t0 + wv < t1) {
        Tile<D> cur = load_tile<D>(region, at(t0 + wv));
        for (int i = t0 + wv; i < t1; i += 4) {
            const int tile = at(i);
            const Tile<D> next = load_tile<D>(region, at(min(i + 4, t1 - 1)));
            const bool edge = tile * 32 < full0 || tile * 32 + 31 > full1;
            tile_step<D, NQ>(cur, region + (size_t)tile * kv4_tile_bytes(D), tile * 32, edge, qf, sight, scale2, st);
            cur = next;
        }
    }
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        if (rho0 + c * 16 >= rows) break;
        if (c) __syncthreads();
        float l = st.l[c];
        l += xor16(l);
        l += xor32(l);
        uint32_t bad = st.bad[c];
        bad |= (uint32_t)__shfl_xor((int)bad, 16);
        bad |= (uint32_t)__shfl_xor((int)bad, 32);
        if (g == 0) { ms[wv][nn] = st.m[c]; ls[wv][nn] = l; bs[wv][nn] = bad; }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < D / 16; i += 4) {
                const f32x4 o = {st.o[c][i][r], st.o[c][i + 1][r], st.o[c][i + 2][r], st.o[c][i + 3][r]};
                *(f32x4*)&os[wv][nn][(4 * g + r) * (D / 16) + i] = o;
            }
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * (D / 4); e += 256) {
            const int n0 = e / (D / 4), d = e % (D / 4) * 4, rho = rho0 + c * 16 + n0;
            if (rho >= rows) break;
            const float m = fmaxf(fmaxf(ms[0][n0], ms[1][n0]), fmaxf(ms[2][n0], ms[3][n0]));
            const float mz = m == -INFINITY ? 0.f : m;
            float sum = 0.f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(ms[w][n0] - mz);
                sum += f * ls[w][n0];
                o += f * *(const f32x4*)&os[w][n0][d];
            }
            if (((bs[0][n0] | bs[1][n0] | bs[2][n0] | bs[3][n0]) >> (d / 32)) & 1) o *= __uint_as_float(0x7fc00000u);
            const int t = rho / group, hq = h * group + rho - t * group;
            const long long row = (long long)seq * a.T + t;
            if (splits == 1) {
                o /= sum;
                if (a.gate.p) {
                    const float4 gt = load4(a.gate.p + row * a.gate.row + hq * a.gate.head + d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] *= sigmoid_f((&gt.x)[i]);
                }
                uint2 w;
                w.x = f2bf2(o[0], o[1]);
                w.y = f2bf2(o[2], o[3]);
                *(uint2*)(const_cast<uint16_t*>(a.out.p) + row * a.out.row + hq * a.out.head + d) = w;
            } else {
                float* p = a.part + ((size_t)blockIdx.x * NQ + c) * kSplitRows * (D + 4) + n0 * (D + 4);
                *(f32x4*)(p + d) = o;
                if (d == 0) { p[D] = m; p[D + 1] = sum; }
            }
        }
    }
}

// Joins the splits of the sequences that have more than one: a block per (sequence, kv head, row), a
// thread per four dims, the splits in order.
template <int D, int NQ>
__global__ void __launch_bounds__(64) attn_kv4_join(Kv4Attn a, int row_tiles) {
    const int group = a.q_heads / a.kv_heads, rows = a.T * group;
    const int rho = blockIdx.x % rows, h = blockIdx.x / rows % a.kv_heads, seq = blockIdx.x / (rows * a.kv_heads);
    const int splits = a.first[seq + 1] - a.first[seq], d = threadIdx.x * 4;
    if (splits == 1 || d >= D) return;
    const int rt = rho / (NQ * 16), c = rho % (NQ * 16) / 16, n0 = rho % 16;
    const size_t step = (size_t)row_tiles * a.kv_heads * NQ * kSplitRows * (D + 4);
    const float* p = a.part + (((size_t)a.first[seq] * a.kv_heads + h) * row_tiles + rt) * NQ * kSplitRows * (D + 4) +
                     ((size_t)c * kSplitRows + n0) * (D + 4);
    float m = -INFINITY;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, p[s * step + D]);
    const float mz = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
        const float f = __builtin_amdgcn_exp2f(p[s * step + D] - mz);
        sum += f * p[s * step + D + 1];
        o += f * *(const f32x4*)(p + s * step + d);
    }
    o /= sum;
    const int t = rho / group, hq = h * group + rho - t * group;
    const long long row = (long long)seq * a.T + t;
    if (a.gate.p) {
        const float4 gt = load4(a.gate.p + row * a.gate.row + hq * a.gate.head + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= sigmoid_f((&gt.x)[i]);
    }
    uint2 w;
    w.x = f2bf2(o[0], o[1]);
    w.y = f2bf2(o[2], o[3]);
    *(uint2*)(const_cast<uint16_t*>(a.out.p) + row * a.out.row + hq * a.out.head + d) = w;
}

template <int D>
static hipError_t launch_attn(Kv4Attn& a, int n, hipStream_t st) {
    const int group = a.q_heads / a.kv_heads, rows = a.T * group, nq = rows > 16 ? 2 : 1;
    const int row_tiles = (rows + nq * 16 - 1) / (nq * 16), items = a.kv_heads * row_tiles;
    // splits: enough blocks to fill the card twice over, each of its four waves with a tile at least
    long long tiles = 0;
    for (int i = 0; i < n; ++i) tiles += tile_list(a.pos[i], a.pos[i] + a.T - 1, a.window, a.sinks).count;
    const long long want = std::max<long long>(1, 512 / items);
    const int per = (int)std::max<long long>(4, (tiles + want - 1) / want);
    int z = 0;
    bool joined = false;
    for (int i = 0; i < n; ++i) {
        a.first[i] = (uint16_t)z;
        const int count = tile_list(a.pos[i], a.pos[i] + a.T - 1, a.window, a.sinks).count;
        const int room = (int)((kMaxSplits / ((long long)items * nq) - z) - (n - 1 - i));
        const int s = std::max(1, std::min(room, (count + per - 1) / per));
        joined |= s > 1;
        z += s;
    }
    a.first[n] = (uint16_t)z;
    const unsigned blocks = (unsigned)z * items;
    if (nq == 1) hipLaunchKernelGGL((attn_kv4_kernel<D, 1>), dim3(blocks), dim3(256), 0, st, a, n, row_tiles);
    else hipLaunchKernelGGL((attn_kv4_kernel<D, 2>), dim3(blocks), dim3(256), 0, st, a, n, row_tiles);
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess || !joined) return rc;
    const unsigned jb = (unsigned)n * a.kv_heads * rows;
    if (nq == 1) hipLaunchKernelGGL((attn_kv4_join<D, 1>), dim3(jb), dim3(64), 0, st, a, row_tiles);
    else hipLaunchKernelGGL((attn_kv4_join<D, 2>), dim3(jb), dim3(64), 0, st, a, row_tiles);
    return hipGetLastError();
}
hipError_t launch_attn_kv4(Kv4Attn& a, int n, hipStream_t st) {
    return a.D == 256 ? launch_attn<256>(a, n, st) : a.D == 128 ? launch_attn<128>(a, n, st) : launch_attn<64>(a, n, st);
}

}  // namespace q35
