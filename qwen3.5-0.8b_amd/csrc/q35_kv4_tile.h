// The steps of attention over the 4-bit cache, for the kernels that differ in which rows and slots meet (q35_kv4.hip,
// q35_kv4_shared.hip): a tile of 32 slots in registers, its fragments, and a wave's running softmax over tiles.
#pragma once
#include "q35_common.h"
#include "q35_kv4.h"

namespace q35 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((__vector_size__(8 * sizeof(float)))) float f32x8;

// The pair of values in byte SEL of w, times the power of two in `scale`'s exponent: exact; NaN
// where that exponent is 255 (all 256 bytes x scales 0 to 252 and 255 compared on MI355X).
template <int SEL>
__device__ __forceinline__ uint32_t two_values(uint32_t w, float scale) {
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

template <int D>
struct Tile {
    u32x4 k[D / 64], v[D / 64];
    uint32_t ks;
    u32x2 vs;
};
// A lane's places in a tile; with the tile's address in scalar registers (scalar_ptr) a load needs no other
// vector register for its address.
struct Lanes { uint32_t blob, ks, vs; };
template <int D>
__device__ __forceinline__ Lanes lane_offsets() {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    return {(uint32_t)lane * 16, (uint32_t)(D == 256 ? lane * 4 : D == 64 ? ((g >> 1) * 16 + m) * 2 : lane * 2),
            (uint32_t)(m * D / 512 * 32 + g * 8)};
}
typedef const __attribute__((address_space(1))) char* gptr;
__device__ __forceinline__ gptr scalar_ptr(const uint8_t* p) {
    const unsigned long long u = (unsigned long long)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return (gptr)(((unsigned long long)hi << 32) | lo);
}
template <class T, bool ONCE = false>
__device__ __forceinline__ T load_at(gptr p, uint32_t off) {
    const auto* w = (const __attribute__((address_space(1))) T*)(p + off);
    if constexpr (ONCE) return __builtin_nontemporal_load(w);
    else return *w;
}
// ONCE: the tile is read by one block only (nontemporal loads)
template <int D, bool ONCE>
__device__ __forceinline__ void load_k(Tile<D>& t, const uint8_t* tile, const Lanes& o) {
    const gptr p = scalar_ptr(tile);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) t.k[i] = load_at<u32x4, ONCE>(p, o.blob + i * 1024);
    const gptr ps = scalar_ptr(tile + 32 * D);
    t.ks = D == 256 ? load_at<uint32_t>(ps, o.ks) : load_at<uint16_t>(ps, o.ks);
}
template <int D, bool ONCE>
__device__ __forceinline__ void load_v(Tile<D>& t, const uint8_t* tile, const Lanes& o) {
    const gptr p = scalar_ptr(tile + 16 * D);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) t.v[i] = load_at<u32x4, ONCE>(p, o.blob + i * 1024);
    t.vs = load_at<u32x2>(scalar_ptr(tile + 33 * D), o.vs);
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

// Entry i of 256 that a wave holds four a lane.
__device__ __forceinline__ int entry(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int i) {
    const uint32_t v = (i & 3) == 0 ? a : (i & 3) == 1 ? b : (i & 3) == 2 ? c : d;
    return __builtin_amdgcn_readlane((int)v, i >> 2);
}

// Which slots a row sees: (pos - window, pos] and [0, sinks); window 0: [0, pos].
struct Sight { int pos, low, sinks; };
__device__ __forceinline__ bool sees(const Sight& s, int slot) { return (slot <= s.pos) & ((slot >= s.low) | (slot < s.sinks)); }

// The running state of NQ x 16 rows over the tiles of one wave.
template <int D, int NQ>
struct Rows {
    float m[NQ];                 // of row n: the reference of its exponents (log2 units)
    f32x4 l[NQ];                 // its sum of weights, four times
    uint32_t bad[NQ];            // groups of 32 dims whose V held a NaN at a slot the row sees
    f32x4 o[NQ][D / 16];         // O^T: dims (4 g + r) D / 16 + i of row n in o[.][i][r]
};

// q: the rows' Q^T operands, [NQ][D / 32], in registers (NQ = 1) or, 16 rows more, in LDS with 64 lanes each
// (the four waves of a block have the same rows). t's registers take the tile at next_p as soon as its K, then its
// V, is used up. TIGHT: 32 rows of 256 dims leave no register for fragments made far ahead.
// edge: some row may not see some slot. FAR: a score times scale2 is rounded before the reference is taken off, and the
// reference lies 28 above the maximum it was taken from, so that weights stay under 2^-20 and 2^18 slots' sum of
// them times the largest V is still a float32 (from references of 2^29 on their spacing takes the 28 in).
template <int D, int NQ, bool ONCE, bool TIGHT, bool FAR, class Q>
__device__ __forceinline__ void tile_step(Tile<D>& t, const uint8_t* tile_p, const uint8_t* next_p, const Lanes& lo, int slot0,
                                          bool edge, const Q& q, const Sight* sight, float scale2, Rows<D, NQ>& st) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    f32x4 s[NQ][2];
#pragma unroll
    for (int c = 0; c < NQ; ++c) s[c][0] = s[c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    q35_bf16x8 qn[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) qn[c] = q(c, 0);
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
        q35_bf16x8 qk[NQ];
#pragma unroll
        for (int c = 0; c < NQ; ++c) { qk[c] = qn[c]; if (k + 1 < D / 32) qn[c] = q(c, k + 1); }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const q35_bf16x8 kf = k_frag<D>(t, half, k);
#pragma unroll
            for (int c = 0; c < NQ; ++c)
                s[c][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qk[c], s[c][half], 0, 0, 0);
        }
        if (TIGHT) __builtin_amdgcn_sched_barrier(0);
    }
    load_k<D, ONCE>(t, next_p, lo);
    u32x2 vsb = t.vs;
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
        float top = fmaxf(fmaxf(s[c][0][0], s[c][0][1]), fmaxf(s[c][0][2], s[c][0][3]));
        top = fmaxf(top, fmaxf(fmaxf(s[c][1][0], s[c][1][1]), fmaxf(s[c][1][2], s[c][1][3])));
        // the reference of the row's exponents follows its maximum only when that is past it by 2^8: weights
        // stay under 2^8 (as exact as under 1), and almost every tile goes without the four lanes' common
        // maximum and the rescale of O
        constexpr float kRoom = FAR ? 28.f : 0.f;
        if (__any(top * scale2 > st.m[c] + (8.f - kRoom))) {
            top = fmaxf(top, xor16(top));
            top = fmaxf(top, xor32(top)) * scale2;
            if (FAR) top += kRoom;
            const float mn = fmaxf(st.m[c], top), al = __builtin_amdgcn_exp2f(st.m[c] - (mn == -INFINITY ? 0.f : mn));
            st.l[c] *= al;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) st.o[c][i] *= al;
            st.m[c] = mn;
        }
        const float ms = st.m[c] == -INFINITY ? 0.f : st.m[c];      // nothing seen so far: e^(-inf) stays 0
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = s[c][j >> 2][j & 3];
            p[j] = __builtin_amdgcn_exp2f(FAR ? x * scale2 - ms : __builtin_fmaf(x, scale2, -ms));
        }
        // Weights rounded to bf16 (2^-8 at most) for the product, as V's values are bf16 and the MFMA takes one type: a
        // float32 product has a sixteenth of its rate. Their sum is that of the rounded ones, a product with ones. Against 64
        // bits outputs are off by 0.0021 to 0.0023 of their size, of which the last rounding alone makes 0.0017.
        const f32x8 pw = {p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
        pf[c] = __builtin_convertvector(pw, q35_bf16x8);     // not f2bf2: the compiler must see what an MFMA is about to read
        st.l[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(q35_bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}),
                                                          pf[c], st.l[c], 0, 0, 0);
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
            if (TIGHT) __builtin_amdgcn_sched_barrier(0);
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
    load_v<D, ONCE>(t, next_p, lo);
}

// Tiles in registers: one of 256 dims (a second one's registers cost more than its loads in flight bring: 128
// lanes x 3 rows x 2000 slots 25.7 instead of 23.8 us), two smaller ones (64 lanes of 128 dims under a
// window 12.9 instead of 14.9 us).
template <int D>
constexpr int kAhead = D == 256 ? 1 : 2;
// W waves take every W-th of the tiles t0 .. t1 - 1 (a block's waves; 1: a wave for itself): the loads of a wave's first ones.
template <int D, int NQ, int W, class TileAt>
__device__ __forceinline__ void first_tiles(Tile<D>* buf, int t0, int t1, const TileAt& tile_at, const Lanes& lo) {
    const int wv = W > 1 ? threadIdx.x >> 6 : 0;
    if (t0 + wv < t1) {
#pragma unroll
        for (int b = 0; b < kAhead<D>; ++b) {
            load_k<D, NQ == 1>(buf[b], tile_at(min(t0 + wv + W * b, t1 - 1)), lo);
            load_v<D, NQ == 1>(buf[b], tile_at(min(t0 + wv + W * b, t1 - 1)), lo);
        }
    }
}
template <int D, int NQ, int W, bool FAR, class At, class TileAt, class Q>
__device__ __forceinline__ void walk_once(Rows<D, NQ>& st, Tile<D>* buf, int t0, int t1, const At& at, const TileAt& tile_at,
                                          const Lanes& lo, const Q& q, int& qlane, const Sight* sight, int full0, int full1,
                                          float scale2) {
    const int wv = W > 1 ? threadIdx.x >> 6 : 0;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        st.m[c] = -INFINITY;
        st.l[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        st.bad[c] = 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) st.o[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int i0 = __builtin_amdgcn_readfirstlane(t0 + wv); i0 < t1; i0 += W * kAhead<D>) {
#pragma unroll
        for (int b = 0; b < kAhead<D>; ++b) {
            const int i = i0 + W * b;
            if (i >= t1) break;
            if (NQ > 1) asm volatile("" : "+v"(qlane));     // or the compiler reads Q ahead of the loop, and spills it
            const int tile = at(i);
            const bool edge = tile * 32 < full0 || tile * 32 + 31 > full1;
            tile_step<D, NQ, NQ == 1, NQ == 2 && D == 256, FAR>(buf[b], tile_at(i), tile_at(min(i + W * kAhead<D>, t1 - 1)), lo,
                                                                tile * 32, edge, q, sight, scale2, st);
        }
    }
}
// A wave's state over its tiles. at(i): the number of the i-th tile (slots 32 at(i) .. + 31), tile_at(i): its address; every
// row sees every slot of the tiles within full0 .. full1.
template <int D, int NQ, int W, class At, class TileAt, class Q>
__device__ __forceinline__ void walk_tiles(Rows<D, NQ>& st, Tile<D>* buf, int t0, int t1, const At& at, const TileAt& tile_at,
                                           const Lanes& lo, const Q& q, int& qlane, const Sight* sight, int full0, int full1,
                                           float scale2) {
    walk_once<D, NQ, W, false>(st, buf, t0, t1, at, tile_at, lo, q, qlane, sight, full0, full1, scale2);
    // Two kinds of rows want their tiles gone over again in the FAR form (the other one is the faster: a 4096-row
    // prompt 83.6 us a call, with a test of the reference in every tile 86.3). References of 2^24 and more: there float32
    // numbers lie 2 and more apart, and the part of a product that its reference was rounded by, which a fused step
    // keeps, is an exponent of its own (past 2^31 it can leave float32). And sums of 2^100 and more, or none any longer:
    // what the waves and the splits (2^10 at most) add up from smaller ones stays a float32.
    bool far = false;
    float big = 0.f;                 // (a NaN anywhere makes it one)
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        far |= __any(fabsf(st.m[c]) >= 16777216.f && st.m[c] != -INFINITY);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) big = __builtin_elementwise_maximum(big, fabsf(st.o[c][i][r]));
    }
    far |= __any(!(big < 0x1p100f));
    if (far) {
        first_tiles<D, NQ, W>(buf, t0, t1, tile_at, lo);
        walk_once<D, NQ, W, true>(st, buf, t0, t1, at, tile_at, lo, q, qlane, sight, full0, full1, scale2);
    }
}
// The W waves' states of `rows` rows: wave w ends a W-th of the row's dims, which the others pass it through LDS, and picks its
// own part out of its registers (through LDS too that was slower: a prompt of 4096 rows 84.2 for 83.4 us, 256 answers to
// 32,768 slots 86.3 for 84.9); a lane keeps its row, and its accumulators go as they are. place(c) gives where row
// 16 c + lane % 16 goes: a function of
// (sums x[r][i] of dim first_dim(r) + i, r < 4, i < D / 16 / W; the reference; the sum of weights).
template <int D, int W>
__device__ __forceinline__ int first_dim(int r) {
    return (4 * ((threadIdx.x & 63) >> 4) + r) * (D / 16) + (threadIdx.x >> 6) * (D / 16 / W);
}
template <int D, int NQ, int W, class Place>
__device__ __forceinline__ void join_waves(Rows<D, NQ>& st, int rows, f32x4 (*os)[W][D / 16 / W][64], float (*ms)[16],
                                           float (*ls)[16], uint32_t (*bs)[16], const Place& place) {
    constexpr int kPart = D / 16 / W;        // of the D / 16 accumulators of 16 rows
    const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, nn = lane & 15, g = lane >> 4;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        if (c * 16 >= rows) break;
        if (NQ > 1 || c) lds_barrier();          // os was read: Q, or the 16 rows before these
        uint32_t bad = st.bad[c];
        bad |= (uint32_t)__shfl_xor((int)bad, 16);
        bad |= (uint32_t)__shfl_xor((int)bad, 32);
        if (g == 0) { ms[wv][nn] = st.m[c]; ls[wv][nn] = st.l[c][0]; bs[wv][nn] = bad; }
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int i = 0; i < kPart; ++i)
                if (w != wv) os[w][wv][i][lane] = st.o[c][w * kPart + i];
        lds_barrier();
        float m = st.m[c], sum = 0.f, f[W];
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, ms[w][nn]);
        bad = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            f[w] = __builtin_amdgcn_exp2f(ms[w][nn] - (m == -INFINITY ? 0.f : m));
            sum += f[w] * ls[w][nn];
            bad |= bs[w][nn];
        }
        f32x4 o[kPart];
#pragma unroll
        for (int i = 0; i < kPart; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w)              // in the same order in every wave
#pragma unroll
            for (int i = 0; i < kPart; ++i) {
                f32x4 v;
                if (w == wv) {
                    v = st.o[c][i];
#pragma unroll
                    for (int k = 1; k < W; ++k) v = wv == k ? st.o[c][k * kPart + i] : v;
                } else {
                    v = os[wv][w][i][lane];
                }
                o[i] += f[w] * v;
            }
        if (c * 16 + nn >= rows) continue;
        float x[4][kPart];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < kPart; ++i)
                x[r][i] = (bad >> (first_dim<D, W>(r) / 32)) & 1 ? __uint_as_float(0x7fc00000u) : o[i][r];
        place(c)(x, m, sum);
    }
}

// Where a row's dims go: normalised, gated, rounded. N dims (1, 2, 4 or 8) from d on.
struct Out {
    const uint16_t* gate;
    uint16_t* out;
    template <class Args>
    __device__ __forceinline__ Out(const Args& a, long long row, int hq) {
        gate = a.gate.p + row * a.gate.row + hq * a.gate.head;
        out = const_cast<uint16_t*>(a.out.p) + row * a.out.row + hq * a.out.head;
    }
    template <int N, class Args>
    __device__ __forceinline__ void store(const Args& a, float* x, float sum, int d) const {
        const float inv = __builtin_amdgcn_rcpf(sum);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= inv;
        if (a.gate.p) {              // sigmoid by the instructions' 2^x and 1/x (a float32 ulp each)
            uint16_t gt[N];
            __builtin_memcpy(gt, gate + d, 2 * N);
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[i] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(bf2f(gt[i]) * -1.44269504088896f));
        }
        uint16_t w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = f2bf(x[i]);
        __builtin_memcpy(out + d, w, 2 * N);
    }
};

}  // namespace q35
