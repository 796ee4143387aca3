// Head norms with rotation, the 4-bit K/V cache, and the attention that reads it.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "q35_kv4_tile.h"

namespace q35 {

__device__ __forceinline__ f32x4 wide(uint2 w) {          // four bf16
    return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                 __uint_as_float(w.y & 0xffff0000u)};
}

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
// 2^x for x <= 0 by the Taylor series of 2^f, |f| <= 1/2 (the first term left out is below 2^-56).
__device__ __forceinline__ double exp2_d(double x) {
    const double k = rint(x), f = (x - k) * 0.69314718055994530942;
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, f, 1.0 / 479001600.0);
    p = __builtin_fma(p, f, 1.0 / 39916800.0);
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(__builtin_fma(p, f, 1.0), (int)k);
}
// cos and sin of pos * theta^(-2 i / rot) = pos * 2^(i * rate). In turns the whole part drops out exactly,
// so a far position keeps its angle: float32 angles are off by up to 4e-3 at position 1e5.
__device__ __forceinline__ float2 turn(int pos, int i, double rate) {
    constexpr double kInv2Pi = 0.15915494309189533577;
    double u = (double)pos * (exp2_d(i * rate) * kInv2Pi);
    u -= rint(u);
    const double q = rint(4.0 * u);
    double s, c;
    sincos_small((u - 0.25 * q) * 6.283185307179586477, s, c);
    const int k = (int)q & 3;
    const double cc = k & 1 ? -s : c, ss = k & 1 ? c : s;
    return k & 2 ? make_float2((float)-cc, (float)-ss) : make_float2((float)cc, (float)ss);
}

// The position of pair `i` of a row, on the pair's axis: all axes' are loaded with the map in flight, not behind it.
__device__ __forceinline__ int axis_position(const AxisHeadArgs& a, int r, int i) {
    const int32_t* p = a.axis_pos + r * a.row_step;
    int at[kAxes];
#pragma unroll
    for (int x = 0; x < kAxes; ++x) at[x] = x < a.axes ? p[a.axis_at[x]] : 0;
    const uint32_t axis = (a.axis_of[i >> 4] >> 2 * (i & 15)) & 3u;
    return axis == 0 ? at[0] : axis == 1 ? at[1] : axis == 2 ? at[2] : at[3];
}

// Sum over a head's 16 lanes in float64, by DPP moves.
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const unsigned long long w = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)w, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(w >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double head_sum(double v) {
    v += dpp_d<0x128>(v);
    v += dpp_d<0x124>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0xB1>(v);
    return v;
}
constexpr int kAngles = 512;         // of a block's rows: kBlockRows x 128
// 1 / sqrt(x) from the instruction's approximation by two Newton steps (float64 to its last bits; NaN of an
// infinity, whose steps are inf * 0)
__device__ __forceinline__ double rsqrt_d(double x) {
    double y = __builtin_amdgcn_rsq(x);
    y = y * __builtin_fma(-0.5 * x * y, y, 1.5);
    return y * __builtin_fma(-0.5 * x * y, y, 1.5);
}

// A block takes `per_block` rows (of few rows with many heads: a part of one row's heads). Its work is the list of
// the rows' (row, head)s of q, then of k, then of v; a wave takes four of one kind at a time, 16 lanes a
// head, a lane dims 64 c + 4 l .. + 3 of each 64: a head's sum needs four steps between lanes for D
// products, and loads and stores are whole 128-byte runs. The rows' angles are made once for the block, with
// the first heads' loads in flight. What the kernel writes is decided by borders (a code's midpoints, a
// scale's step), so every float32 operation is one rounding in the stated order, and the sum of
// squares, the root and the angles are float64. QUADS: rot / 2 is a multiple of 4, so a lane's four dims lie
// on one side of the pairs. TINY: eps is so small (under 2^-250) that a root may pass float32; without that form's care
// 1999 rows as below take 0.4 us less.
// Many rows: memory and the instructions a head takes share the time (4096 rows of 8 + 2 heads of 256, 42 MB: 11.2 us,
// the VALU at work in 65 % of the CUs' busy cycles; 1999 rows of 32 + 2 x 8 heads of 128 with the append, 51 MB:
// 14.9 us, 75 %, its codes in stores of 2 bytes a lane that the cache's fragment order scatters); few rows: the chain
// of launch, loads and angles (1 row 3.5 us, 256 rows with the append 5.5).
constexpr int kBlockRows = 4;
template <int D, bool QUADS, bool TINY, class Args>
__global__ void __launch_bounds__(256) heads_kernel(Args a, int rows, int per_block, int parts, int some) {
    constexpr bool kOnAxes = std::is_same<Args, AxisHeadArgs>::value;
    constexpr int C = D / 64;
    __shared__ float xs[4][4][D];
    __shared__ float2 cs[kAngles];
    __shared__ int2 at[kBlockRows];          // a row's position and lane
    const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, j = lane >> 4, l = lane & 15;
    const int r0 = blockIdx.x / parts * per_block, nr = min(per_block, rows - r0), half = a.rot / 2;
    // wave items of each kind, and this block's part of them
    const int iq = a.q.p ? (nr * a.q_heads + 3) / 4 : 0, ik = (nr * a.kv_heads + 3) / 4;
    const int i0 = blockIdx.x % parts * some, i1 = min(i0 + some, iq + (a.v.p ? 2 : 1) * ik);
    struct Item { int kind, rr, h; bool on; };
    const auto item = [&](int i) {
        Item t;
        t.kind = i < iq ? 0 : i < iq + ik ? 1 : 2;
        const int heads = t.kind == 0 ? a.q_heads : a.kv_heads, x = (t.kind == 0 ? i : t.kind == 1 ? i - iq : i - iq - ik) * 4 + j;
        t.rr = heads == 1 ? x : (int)__umulhi((uint32_t)x, t.kind == 0 ? a.q_inv : a.kv_inv);
        t.h = x - t.rr * heads;
        t.on = i < i1 && t.rr < nr;
        return t;
    };
    const auto fetch = [&](const Item& t, uint2* w) {
        const HeadView& in = t.kind == 0 ? a.q : t.kind == 1 ? a.k : a.v;
        const uint16_t* p = in.p + (r0 + t.rr) * in.row + t.h * in.head + 4 * l;
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = t.on ? *(const uint2*)(p + 64 * c) : make_uint2(0, 0);
    };
    Item now = item(__builtin_amdgcn_readfirstlane(i0 + wv));
    uint2 raw[C];
    fetch(now, raw);
    for (int i = tid; i < nr * half; i += 256) {
        const int rr = i / half, r = r0 + rr;
        if constexpr (kOnAxes) cs[i] = turn(axis_position(a, r, i - rr * half), i - rr * half, a.rate);
        else cs[i] = turn(a.pos[r / a.T] + r % a.T, i - rr * half, a.rate);
    }
    if (tid < nr) {
        const int r = r0 + tid, seq = r / a.T;
        at[tid] = make_int2(a.pos[seq] + r - seq * a.T, a.lane[seq]);
    }
    lds_barrier();
    for (int i = __builtin_amdgcn_readfirstlane(i0 + wv); i < i1; i += 4) {      // whole waves; no block barrier in the loop
        const Item t = now;
        const int kind = t.kind;
        f32x4 x[C];
#pragma unroll
        for (int c = 0; c < C; ++c) x[c] = wide(raw[c]);
        now = item(i + 4);
        fetch(now, raw);
        if (kind < 2) {
            const uint16_t* nw = (kind == 0 ? a.q_norm : a.k_norm) + 4 * l;
            uint2 w[C];
#pragma unroll
            for (int c = 0; c < C; ++c) w[c] = *(const uint2*)(nw + 64 * c);
            double ss = 0.0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = __builtin_fma((double)x[c][e], (double)x[c][e], ss);
            const double mean = head_sum(ss) * (1.0 / D) + a.eps, root = rsqrt_d(mean);
            float rs = (float)root;
            if (mean == INFINITY) rs = 0.f;
            if (TINY) {                      // of subnormal numbers 2^64 of it go to x first, exactly
                const bool past = rs == INFINITY;
                if (past) rs = (float)(root * 0x1p-64);
#pragma unroll
                for (int c = 0; c < C; ++c) x[c] *= past ? 0x1p64f : 1.f;
            }
            float* hx = xs[wv][j];
            wave_sync();
#pragma unroll
            for (int c = 0; c < C; ++c) {
                x[c] = x[c] * rs * (1.0f + wide(w[c]));
                if (64 * c < a.rot) *(f32x4*)&hx[64 * c + 4 * l] = x[c];
            }
            wave_sync();
            const float2* cr = cs + (t.on ? t.rr : 0) * half;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int d = 64 * c + 4 * l;
                if (64 * c >= a.rot) break;
                if (QUADS) {
                    if (d < a.rot) {
                        const bool low = d < half;
                        const int k = low ? d : d - half;
                        const f32x4 o = *(const f32x4*)&hx[low ? d + half : k];
                        const f32x4 c0 = *(const f32x4*)&cr[k], c1 = *(const f32x4*)&cr[k + 2];
                        const f32x4 p = x[c] * f32x4{c0[0], c0[2], c1[0], c1[2]}, q = o * f32x4{c0[1], c0[3], c1[1], c1[3]};
                        x[c] = low ? p - q : p + q;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (d + e < half) {
                            const float2 cc = cr[d + e];
                            x[c][e] = x[c][e] * cc.x - hx[d + e + half] * cc.y;
                        } else if (d + e < a.rot) {
                            const float2 cc = cr[d + e - half];
                            x[c][e] = x[c][e] * cc.x + hx[d + e - half] * cc.y;
                        }
                    }
                }
            }
        }
        const HeadView& out = kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out;
        uint16_t* op = const_cast<uint16_t*>(out.p) + (r0 + t.rr) * out.row + t.h * out.head + 4 * l;
        if (kind == 0 || !a.cache) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (t.on) *(uint2*)(op + 64 * c) = make_uint2(f2bf2(x[c][0], x[c][1]), f2bf2(x[c][2], x[c][3]));
            continue;
        }
        const int2 where = at[t.on ? t.rr : 0];
        uint8_t* tile = a.cache + where.y * a.lane_bytes + t.h * a.region + (size_t)(where.x >> 5) * kv4_tile_bytes(D);
        const int tk = where.x & 31;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            // the group's largest magnitude as bits (8 lanes): an infinity or a NaN is the largest of all
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[c][e]) & 0x7fffffffu);
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xf, 0xf, false));   // lane 7 - i of 8
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
            // top = 1.m 2^E: 6 * 2^(E - 2) covers it up to m = 0.5, else one step more. Kept within
            // 2^-119 .. 2^125, so that no value overflows bf16 or loses bits below its normal range.
            uint32_t b = max((int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u), 8);
            b = top >= 0x7f800000u ? 255u : min(b, 252u);
            const float sc = scale_of(b);
            uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[c][0], x[c][1], sc, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[c][2], x[c][3], sc, 1);
            const int d = 64 * c + 4 * l;
            if (!t.on) continue;
            if (out.p) *(uint2*)(op + 64 * c) = make_uint2(two_values<0>(code, sc), two_values<1>(code, sc));
            *(uint16_t*)(tile + (kind == 1 ? kv4_k_code(D, tk, d) : kv4_v_code(D, tk, d))) = (uint16_t)code;
            if ((l & 7) == 0) tile[kind == 1 ? kv4_k_scale(D, tk, d >> 5) : kv4_v_scale(D, tk, d >> 5)] = (uint8_t)b;
        }
    }
}

template <class Args>
static hipError_t launch(Args& a, int n, hipStream_t st) {
    const int rows = n * a.T, kinds = a.v.p ? 2 : 1;
    // rows of a block: two when that leaves every CU two blocks or more, four when it leaves every CU four (1999 rows of
    // 32 q heads by one 16.4 us, two 15.8, four 19.7; 4096 of 8 by one 17.1, two 14.2, four 12.1: both lines lie between
    // these two shapes, and the number of heads is not in them); of very few rows with many heads, four wave
    // items (one a wave) in a block
    const int per_block = rows >= 4096 ? kBlockRows : rows >= 1024 ? 2 : 1;
    const int items = ((a.q.p ? per_block * a.q_heads + 3 : 0) / 4) + kinds * ((per_block * a.kv_heads + 3) / 4);
    const int some = rows < 256 ? std::min(items, 4) : items, parts = (items + some - 1) / some;
    const long long blocks = (long long)((rows + per_block - 1) / per_block) * parts;
    if (blocks > kLaunchBlocks) return hipErrorInvalidValue;
    a.q_inv = a.q_heads > 1 ? (uint32_t)(0x100000000ull / a.q_heads + 1) : 0;
    a.kv_inv = a.kv_heads > 1 ? (uint32_t)(0x100000000ull / a.kv_heads + 1) : 0;
    const bool quads = a.rot % 8 == 0;
    const auto pick = [&](auto tiny) {
        constexpr bool t = decltype(tiny)::value;
        return a.D == 256 ? (quads ? heads_kernel<256, true, t, Args> : heads_kernel<256, false, t, Args>)
             : a.D == 128 ? (quads ? heads_kernel<128, true, t, Args> : heads_kernel<128, false, t, Args>)
                          : (quads ? heads_kernel<64, true, t, Args> : heads_kernel<64, false, t, Args>);
    };
    const auto k = a.eps < 0x1p-250 ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, a, rows, per_block, parts, some);
    return hipGetLastError();
}
hipError_t launch_heads(HeadArgs& a, int n, hipStream_t st) { return launch(a, n, st); }
hipError_t launch_heads(AxisHeadArgs& a, int n, hipStream_t st) { return launch(a, n, st); }

// ------------------------------------------------------------------ rows in and out of the cache
// A thread per 8 dims of a (lane, kv head, slot): 4 bytes of codes, and a scale byte in one of four. Copies between
// the fragment order and rows, for snapshots and checks: no step's path has it, so it is left simple.
template <bool WRITE>
__global__ void __launch_bounds__(256) kv4_copy_kernel(Kv4Copy a, long long block0) {
    const int per = a.D / 8;
    const long long i = (block0 + blockIdx.x) * 256 + threadIdx.x;
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
            if (WRITE) *c = *o > 252 ? 255 : *o;     // (2^126 and up: past bf16)
            else *o = *c;
        }
    }
}
hipError_t launch_kv4_copy(const Kv4Copy& a, bool write, hipStream_t st) {
    const long long n = (long long)a.n_lanes * a.kv_heads * a.n_slots * (a.D / 8), blocks = (n + 255) / 256;
    for (long long b = 0; b < blocks; b += kLaunchBlocks) {
        const dim3 grid((unsigned)std::min<long long>(kLaunchBlocks, blocks - b));
        if (write) hipLaunchKernelGGL(kv4_copy_kernel<true>, grid, dim3(256), 0, st, a, b);
        else hipLaunchKernelGGL(kv4_copy_kernel<false>, grid, dim3(256), 0, st, a, b);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

// ------------------------------------------------------------------ attention
// Rows of one sequence and kv head: the T new rows times the head's `group` query heads, row rho =
// t * group + g at position pos + t. S^T = K Q^T and O^T = V^T P^T on 16x16x32 bf16 MFMAs with the
// slots (S^T) and the dims (O^T) in M and 16 rows in N: a lane's column is one row in both, so the row's
// maximum, sum and rescale live in the lane, and S^T's accumulators are P^T's operand as they are.
// Decode and verify rows are bound by the cache's bytes: 256 lanes x 4096 slots of 2 heads of 256 (574 MB) 88 us,
// 6.5 TB/s; 128 lanes x 3 rows x up to 2000 slots (84 MB) 23 us and a join of 4, a block a CU or two for 40 tiles.
// Prompts are bound by what the VALU issues beside the MFMAs, most of it making bf16 fragments of codes (192 of a
// step's 293 instructions for 66 MFMAs of 32 rows): 4096 rows of 8 heads of 256 (69 GFLOP) 85 us, 8192 rows 279 (985
// TFLOP/s; a library's 8192^3 product reaches 1191). These are launches back to back; the first ones after a card that
// idled take 98 and 320.
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
constexpr int kSeqSplits = 256;      // splits of one sequence
size_t kv4_part_floats() { return (size_t)kMaxSplits * kSplitRows * (256 + 4); }

// What a block needs of its sequence. The arrays are kernel arguments, cold in every cache at a launch:
// a wave loads all of them at once (four entries a lane) and finds the sequence by counting the entries of
// first[] up to z, instead of bisecting them with a round trip to memory per step.
struct Seq { int i, pos, lane, split, splits; };
__device__ __forceinline__ Seq find_seq(const Kv4Attn& a, int z) {
    const int lane = threadIdx.x & 63;
    const uint2 f = ((const uint2*)a.first)[lane], l = ((const uint2*)a.lane)[lane];
    const uint4 p = ((const uint4*)a.pos)[lane];
    const uint32_t f0 = f.x & 0xffffu, f1 = f.x >> 16, f2 = f.y & 0xffffu, f3 = f.y >> 16, zz = (uint32_t)z;
    const int i = __popcll(__ballot(f0 <= zz)) + __popcll(__ballot(f1 <= zz)) + __popcll(__ballot(f2 <= zz)) +
                  __popcll(__ballot(f3 <= zz)) - 1;
    Seq s;
    s.i = i;
    s.pos = entry(p.x, p.y, p.z, p.w, i);
    s.lane = entry(l.x & 0xffffu, l.x >> 16, l.y & 0xffffu, l.y >> 16, i);
    const int at = entry(f0, f1, f2, f3, i), end = i + 1 < a.n ? entry(f0, f1, f2, f3, i + 1) : a.splits;
    s.split = z - at;
    s.splits = end - at;
    return s;
}

__device__ __forceinline__ Out out_of(const Kv4Attn& a, long long seq, int h, int rho) {
    const int group = a.q_heads / a.kv_heads, t = rho / group;
    return Out(a, seq * a.T + t, h * group + rho - t * group);
}
// Partial result of (split z, kv head h, row rho): D sums, then the maximum and the sum of the weights.
template <int D, int NQ>
__device__ __forceinline__ const float* part_of(const Kv4Attn& a, int row_tiles, int z, int h, int rho) {
    return a.part + ((((size_t)z * a.kv_heads + h) * row_tiles + rho / (NQ * 16)) * NQ * kSplitRows + rho % (NQ * 16)) * (D + 4);
}

// A block per (sequence, split of its tiles, kv head, NQ x 16 rows): its four waves take every fourth tile
// with the next ones' loads in flight, and their states are joined through LDS. Under the causal mask the last
// row tiles are the longest: they come first, so that the short ones fill the CUs' ends (4096 rows of 8 heads of
// 256 in one prompt 96 us, launched with waits between; each block with a long and a short tile in turn 100). One sequence
// of at most two blocks a CU has them all at once: the second of a CU is then short where the first is long (2048
// rows 35 us, without 38, ascending 47; back to back it takes 34).
template <int D, int NQ>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 1) attn_kv4_kernel(Kv4Attn a, int row_tiles) {
    __shared__ f32x4 os[4][4][D / 64][64];
    __shared__ float ms[4][16], ls[4][16];
    __shared__ uint32_t bs[4][16];
    static_assert(NQ == 1 || sizeof(os) >= NQ * (D / 32) * 1024, "the Q operands lie where the waves' sums go at the end");
    const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, nn = lane & 15, g = lane >> 4;
    const int per_split = row_tiles * a.kv_heads, z = blockIdx.x / per_split;
    int ix = blockIdx.x % per_split;
    if (per_split == gridDim.x && per_split <= 512 && ix >= 256) ix = per_split - 1 - (ix - 256);
    const int h = ix % a.kv_heads, rt = row_tiles - 1 - ix / a.kv_heads;
    const Seq sq = find_seq(a, z);
    const int seq = sq.i, splits = sq.splits, pos = sq.pos, group = a.q_heads / a.kv_heads, rows = a.T * group;
    const uint8_t* region = a.cache + sq.lane * a.lane_bytes + h * a.region;
    // positive, so that the largest product has the largest exponent and a dropped one's -inf stays it: a negative
    // scale's sign goes to q, 0 becomes the smallest number there is (the largest product then counts 5e-7)
    const float scale2 = fmaxf(fabsf(a.scale) * 1.44269504088896f, 0x1p-149f);
    const Lanes lo = lane_offsets<D>();
    const int rho0 = rt * NQ * 16, rho1 = min(rho0 + NQ * 16, rows) - 1;
    const TileList tl = tile_list(pos + rho0 / group, pos + rho1 / group, a.window, a.sinks);
    const int t0 = (int)((long long)tl.count * sq.split / splits), t1 = (int)((long long)tl.count * (sq.split + 1) / splits);
    const auto q_at = [&](int rho, int gg, int k) {
        rho = min(rho, rows - 1);
        const int t = rho / group;
        u32x4 w = *(const u32x4*)(a.q.p + ((long long)seq * a.T + t) * a.q.row + (h * group + rho - t * group) * a.q.head +
                                  gg * (D / 4) + 8 * k);
        if (a.scale < 0.f) w ^= 0x80008000u;
        return __builtin_bit_cast(q35_bf16x8, w);
    };
    auto at = [&](int i) { return i < tl.sink ? i : i - tl.sink + tl.main; };
    const auto tile_at = [&](int i) { return region + (size_t)at(i) * kv4_tile_bytes(D); };
    Tile<D> buf[kAhead<D>];
    first_tiles<D, NQ, 4>(buf, t0, t1, tile_at, lo);
    q35_bf16x8 qf[NQ == 1 ? D / 32 : 1];
    q35_bf16x8* ql = (q35_bf16x8*)&os[0][0][0][0];
    if constexpr (NQ == 1) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k) qf[k] = q_at(rho0 + nn, g, k);
    } else {
        for (int i = tid; i < NQ * (D / 32) * 64; i += 256) {
            const int ln = i & 63, k = i / 64 % (D / 32), c = i / (64 * (D / 32));
            ql[i] = q_at(rho0 + c * 16 + (ln & 15), ln >> 4, k);
        }
        lds_barrier();
    }
    int qlane = lane;
    const auto q = [&](int c, int k) { return NQ == 1 ? qf[k] : ql[(c * (D / 32) + k) * 64 + qlane]; };
    Sight sight[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int p = pos + min(rho0 + c * 16 + nn, rows - 1) / group;
        sight[c] = {p, a.window > 0 ? p - a.window + 1 : 0, a.sinks};
    }
    // tiles whose every slot every row of the block sees: from the last row's window to the first row's slot
    const int full0 = a.window > 0 ? max(pos + rho1 / group - a.window + 1, 0) : 0, full1 = pos + rho0 / group;
    Rows<D, NQ> st;
    walk_tiles<D, NQ, 4>(st, buf, t0, t1, at, tile_at, lo, q, qlane, sight, full0, full1, scale2);
    join_waves<D, NQ, 4>(st, rows - rho0, os, ms, ls, bs, [&](int c) {
        const Out to = out_of(a, seq, h, rho0 + c * 16 + nn);
        return [=, &a](float (*x)[D / 64], float m, float sum) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = first_dim<D, 4>(r);
                if (splits == 1) {
                    to.store<D / 64>(a, x[r], sum, d);
                } else {
                    float* p = a.part + ((((size_t)z * a.kv_heads + h) * row_tiles + rt) * NQ + c) * kSplitRows * (D + 4) + nn * (D + 4);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) p[d + i] = x[r][i];
                    if (d == 0) { p[D] = m; p[D + 1] = sum; }
                }
            }
        };
    });
}

// Joins the splits of sequences that have few (up to 8): a thread per four dims of a row, all its
// loads at once. A launch and one trip to memory: 128 lanes x 12 rows of 256 dims 4.3 us.
constexpr int kFewSplits = 8;
template <int D, int NQ>
__global__ void __launch_bounds__(256) attn_kv4_join_few(Kv4Attn a, int row_tiles) {
    const int rows = a.T * (a.q_heads / a.kv_heads);
    const long long e = ((long long)blockIdx.x * 256 + threadIdx.x) / (D / 4);
    const int d = threadIdx.x % (D / 4) * 4;
    const int rho = (int)(e % rows), h = (int)(e / rows % a.kv_heads);
    const long long seq = e / ((long long)rows * a.kv_heads);
    if (seq >= a.n) return;
    const int first = a.first[seq], splits = (seq + 1 < a.n ? a.first[seq + 1] : a.splits) - first;
    if (splits == 1) return;
    const float* p = part_of<D, NQ>(a, row_tiles, first, h, rho);
    const size_t step = (size_t)a.kv_heads * row_tiles * NQ * kSplitRows * (D + 4);
    f32x4 o[kFewSplits];
    float2 ml[kFewSplits];
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        const bool in = s < splits;
        o[s] = in ? *(const f32x4*)(p + s * step + d) : f32x4{0.f, 0.f, 0.f, 0.f};
        ml[s] = in ? *(const float2*)(p + s * step + D) : make_float2(-INFINITY, 0.f);
    }
    float m = ml[0].x;
#pragma unroll
    for (int s = 1; s < kFewSplits; ++s) m = fmaxf(m, ml[s].x);
    const float mz = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        const float f = __builtin_amdgcn_exp2f(ml[s].x - mz);
        sum += f * ml[s].y;
        x += f * o[s];
    }
    out_of(a, seq, h, rho).store<4>(a, (float*)&x, sum, d);
}

// The same for any number of splits: a block per (sequence, kv head, row, 64 dims). The splits' factors are
// made once into LDS; 16 threads take a split's dims, 16 splits at a time, and their sums meet in LDS:
// always in the same order. Latency here too: 8 rows of 128 splits 4.5 us.
template <int D, int NQ>
__global__ void __launch_bounds__(256) attn_kv4_join(Kv4Attn a, int row_tiles) {
    __shared__ float fs[kSeqSplits];
    __shared__ float red[8];
    __shared__ f32x4 os[256];
    const int rows = a.T * (a.q_heads / a.kv_heads), tid = threadIdx.x, d = blockIdx.x % (D / 64) * 64 + tid % 16 * 4;
    const int e = blockIdx.x / (D / 64), rho = e % rows, h = e / rows % a.kv_heads, seq = e / (rows * a.kv_heads);
    const int first = a.first[seq], splits = (seq + 1 < a.n ? a.first[seq + 1] : a.splits) - first;
    if (splits == 1) return;
    const float* p = part_of<D, NQ>(a, row_tiles, first, h, rho);
    const size_t step = (size_t)a.kv_heads * row_tiles * NQ * kSplitRows * (D + 4);
    f32x4 v[kSeqSplits / 16];
#pragma unroll
    for (int i = 0; i < kSeqSplits / 16; ++i) {
        const int s = i * 16 + tid / 16;
        v[i] = s < splits ? *(const f32x4*)(p + s * step + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float2 ml = make_float2(-INFINITY, 0.f);
    if (tid < splits) ml = *(const float2*)(p + tid * step + D);
    const float wm = wave_max(ml.x);
    if ((tid & 63) == 0) red[tid >> 6] = wm;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float f = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
    fs[tid] = f;
    const float ws = wave_sum(f * ml.y);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = ws;
    __syncthreads();
    const float sum = (red[4] + red[5]) + (red[6] + red[7]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kSeqSplits / 16; ++i) o += fs[i * 16 + tid / 16] * v[i];
    os[tid] = o;
    __syncthreads();
    if (tid >= 16) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) o += os[i * 16 + tid];
    out_of(a, seq, h, rho).store<4>(a, (float*)&o, sum, d);
}

template <int D>
static hipError_t launch_attn(Kv4Attn& a, int n, hipStream_t st) {
    const int group = a.q_heads / a.kv_heads, rows = a.T * group, nq = rows > 16 ? 2 : 1;
    const int row_tiles = (rows + nq * 16 - 1) / (nq * 16), items = kv4_attn_items(a.q_heads, a.kv_heads, a.T);
    // splits: a block a CU (two a CU: 64 lanes under a window 15.6 instead of 12.9 us with the join, 100 lanes x 4096
    // slots 50.6 instead of 45.7), each of its four waves with two tiles at least (four: 1 lane x 32768 slots
    // 14.7 instead of 13.6)
    long long tiles = 0;
    for (int i = 0; i < n; ++i) tiles += tile_list(a.pos[i], a.pos[i] + a.T - 1, a.window, a.sinks).count;
    const long long want = std::max<long long>(1, 256 / items);
    const int per = (int)std::max<long long>(8, (tiles + want - 1) / want);
    int z = 0;
    int most = 1;
    for (int i = 0; i < n; ++i) {
        a.first[i] = (uint16_t)z;
        const int count = tile_list(a.pos[i], a.pos[i] + a.T - 1, a.window, a.sinks).count;
        const int room = (int)((kMaxSplits / ((long long)items * nq) - z) - (n - 1 - i));
        const int s = std::max(1, std::min({room, kSeqSplits, (count + per - 1) / per}));
        most = std::max(most, s);
        z += s;
    }
    for (int i = n; i < kSeqArgs; ++i) a.first[i] = 0xffff;
    a.n = n;
    a.splits = z;
    if ((long long)z * items > kLaunchBlocks) return hipErrorInvalidValue;
    const unsigned blocks = (unsigned)z * items;
    if (nq == 1) hipLaunchKernelGGL((attn_kv4_kernel<D, 1>), dim3(blocks), dim3(256), 0, st, a, row_tiles);
    else hipLaunchKernelGGL((attn_kv4_kernel<D, 2>), dim3(blocks), dim3(256), 0, st, a, row_tiles);
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess || most == 1) return rc;
    const long long heads = (long long)n * a.kv_heads * rows;
    if (most <= kFewSplits) {
        const unsigned jb = (unsigned)((heads * (D / 4) + 255) / 256);
        if (nq == 1) hipLaunchKernelGGL((attn_kv4_join_few<D, 1>), dim3(jb), dim3(256), 0, st, a, row_tiles);
        else hipLaunchKernelGGL((attn_kv4_join_few<D, 2>), dim3(jb), dim3(256), 0, st, a, row_tiles);
    } else {
        const unsigned jb = (unsigned)(heads * (D / 64));
        if (nq == 1) hipLaunchKernelGGL((attn_kv4_join<D, 1>), dim3(jb), dim3(256), 0, st, a, row_tiles);
        else hipLaunchKernelGGL((attn_kv4_join<D, 2>), dim3(jb), dim3(256), 0, st, a, row_tiles);
    }
    return hipGetLastError();
}
hipError_t launch_attn_kv4(Kv4Attn& a, int n, hipStream_t st) {
    return a.D == 256 ? launch_attn<256>(a, n, st) : a.D == 128 ? launch_attn<128>(a, n, st) : launch_attn<64>(a, n, st);
}

}  // namespace q35
