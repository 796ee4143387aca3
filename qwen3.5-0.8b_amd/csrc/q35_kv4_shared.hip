// Attention of answers that share long prompts, over the 4-bit cache: a prompt's slots are read once for all of its
// answers.
//
// A row's softmax over its prompt's slots and its own is the join of parts: with a part's reference m_p, sum of weights
// l_p and sums o_p, out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p. A prompt's part has the rows of all its answers
// (answers x T x query heads of a kv head) in the MFMAs' N dimension, so a tile of slots is fetched and turned
// into bf16 once for 32 rows instead of once for each answer's 4 or 16; the answers' own slots are short lists, as in
// the attention of single lanes. Both kinds are blocks of one launch, split so that all take about as long; a second launch
// joins the parts.
#include <algorithm>
#include <climits>

#include "q35_answers.h"
#include "q35_kv4_tile.h"

namespace q35 {

long long kv4_shared_room(int D) { return (long long)(kv4_part_floats() / (D + 4)); }

// What a block works on: rows rho0 .. of the `rows` rows of the sorted sequences from `start` on, over tiles t0 .. t1 - 1.
struct Part {
    const uint8_t* region;
    int start, rows, rho0, h, t0, t1;
    int last;                        // a prompt's last slot; -1: a row sees up to its own position
    int pos;                         // of the sequence's row 0 (own slots)
    long long row0;                  // where the part's rows go in the partial results
};

__device__ __forceinline__ Part prompt_part(const Kv4Shared& a, int per, int tile_rows) {
    const int b = blockIdx.x, lane = threadIdx.x & 63;
    const int f = a.gfirst[lane], pt = a.gpart[lane], ln = a.glen[lane], gl = a.glane[lane], gs = a.gstart[lane], sp = a.gsplits[lane];
    const int j = __popcll(__ballot(f <= b)) - 1;
    const auto of = [&](int v, int i) { return __builtin_amdgcn_readlane(v, i); };
    const int end = j + 1 < a.groups ? of(gs, j + 1) : a.n, splits = of(sp, j), tiles = (of(ln, j) + 31) >> 5;
    // splits vary fastest: the blocks of one split, which read the same tiles, lie on one XCD where the
    // splits are a multiple of 8
    const int ix = b - of(f, j), split = ix % splits, item = ix / splits;
    Part p;
    p.start = of(gs, j);
    p.rows = (end - p.start) * per;
    p.h = item % a.kv_heads;
    p.rho0 = item / a.kv_heads * tile_rows;
    p.t0 = (int)((long long)tiles * split / splits);
    p.t1 = (int)((long long)tiles * (split + 1) / splits);
    p.region = a.prefix + of(gl, j) * a.prefix_lane + p.h * a.prefix_region;
    p.last = of(ln, j) - 1;
    p.pos = 0;
    p.row0 = of(pt, j) + (long long)(split * a.kv_heads + p.h) * p.rows;
    return p;
}
__device__ __forceinline__ Part own_part(const Kv4Shared& a, int per, int tile_rows) {
    const int row_tiles = (per + tile_rows - 1) / tile_rows, lane = threadIdx.x & 63;
    const int b = blockIdx.x - a.prefix_blocks, z = b / (row_tiles * a.kv_heads), ix = b % (row_tiles * a.kv_heads);
    const uint2 f = ((const uint2*)a.first)[lane], l = ((const uint2*)a.lane)[lane];
    const uint4 ps = ((const uint4*)a.pos)[lane];
    const uint32_t f0 = f.x & 0xffffu, f1 = f.x >> 16, f2 = f.y & 0xffffu, f3 = f.y >> 16, zz = (uint32_t)z;
    const int i = __popcll(__ballot(f0 <= zz)) + __popcll(__ballot(f1 <= zz)) + __popcll(__ballot(f2 <= zz)) +
                  __popcll(__ballot(f3 <= zz)) - 1;
    const int first = entry(f0, f1, f2, f3, i), splits = (i + 1 < a.n ? entry(f0, f1, f2, f3, i + 1) : a.own_splits) - first;
    Part p;
    p.start = i;
    p.rows = per;
    p.h = ix % a.kv_heads;
    p.rho0 = ix / a.kv_heads * tile_rows;
    p.pos = entry(ps.x, ps.y, ps.z, ps.w, i);
    const int tiles = ((p.pos + (min(p.rho0 + tile_rows, per) - 1) / (per / a.T)) >> 5) + 1;
    p.t0 = (int)((long long)tiles * (z - first) / splits);
    p.t1 = (int)((long long)tiles * (z - first + 1) / splits);
    p.region = a.cache + entry(l.x & 0xffffu, l.x >> 16, l.y & 0xffffu, l.y >> 16, i) * a.lane_bytes + p.h * a.region;
    p.last = -1;
    p.row0 = a.own_part + (long long)(z * a.kv_heads + p.h) * per;
    return p;
}

// A block's part: its four waves take every fourth tile, their states are joined through LDS.
template <int D, int NQ>
__device__ __forceinline__ void part_rows(const Kv4Shared& a, const Part& p, f32x4 (*os)[4][D / 64][64], float (*ms)[16],
                                          float (*ls)[16], uint32_t (*bs)[16]) {
    const int tid = threadIdx.x, lane = tid & 63, nn = lane & 15, g = lane >> 4;
    const int group = a.q_heads / a.kv_heads, per = a.T * group;
    const float scale2 = fmaxf(fabsf(a.scale) * 1.44269504088896f, 0x1p-149f);      // (as in the attention of single lanes)
    const Lanes lo = lane_offsets<D>();
    const auto at = [&](int i) { return i; };
    const auto tile_at = [&](int i) { return p.region + (size_t)i * kv4_tile_bytes(D); };
    Tile<D> buf[kAhead<D>];
    first_tiles<D, NQ>(buf, p.t0, p.t1, tile_at, lo);
    const uint16_t* qrow[NQ];
    Sight sight[NQ];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int rho = min(p.rho0 + c * 16 + nn, p.rows - 1), i = rho / per, r = rho - i * per, t = r / group;
        qrow[c] = a.q.p + ((long long)a.seq[p.start + i] * a.TT + t) * a.q.row + (p.h * group + r - t * group) * a.q.head;
        sight[c] = {p.last >= 0 ? p.last : p.pos + t, 0, 0};
    }
    const auto q_at = [&](int c, int gg, int k) {
        u32x4 w = *(const u32x4*)(qrow[c] + gg * (D / 4) + 8 * k);
        if (a.scale < 0.f) w ^= 0x80008000u;
        return __builtin_bit_cast(q35_bf16x8, w);
    };
    q35_bf16x8 qf[NQ == 1 ? D / 32 : 1];
    q35_bf16x8* ql = (q35_bf16x8*)&os[0][0][0][0];
    if constexpr (NQ == 1) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k) qf[k] = q_at(0, g, k);
    } else {
        // wave w fetches every fourth step's operands
#pragma unroll
        for (int c = 0; c < NQ; ++c)
            for (int k = tid >> 6; k < D / 32; k += 4) ql[(c * (D / 32) + k) * 64 + lane] = q_at(c, g, k);
        lds_barrier();
    }
    int qlane = lane;
    const auto q = [&](int c, int k) { return NQ == 1 ? qf[k] : ql[(c * (D / 32) + k) * 64 + qlane]; };
    const int full1 = p.last >= 0 ? p.last : p.pos + p.rho0 / group;
    Rows<D, NQ> st;
    walk_tiles<D, NQ>(st, buf, p.t0, p.t1, at, tile_at, lo, q, qlane, sight, 0, full1, scale2);
    join_waves<D, NQ>(st, p.rows - p.rho0, os, ms, ls, bs, [&](int c) {
        float* to = a.part + (p.row0 + p.rho0 + c * 16 + nn) * (D + 4);
        return [=](float* x, int d, float m, float sum) {
#pragma unroll
            for (int i = 0; i < D / 64; ++i) to[d + i] = x[i];
            if (d == 0) { to[D] = m; to[D + 1] = sum; }
        };
    });
}

// NQP, NQO: 16 rows a block takes of a prompt's and of an answer's own.
template <int D, int NQP, int NQO>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 1) shared_kernel(Kv4Shared a) {
    __shared__ f32x4 os[4][4][D / 64][64];
    __shared__ float ms[4][16], ls[4][16];
    __shared__ uint32_t bs[4][16];
    static_assert(NQP == 1 || sizeof(os) >= NQP * (D / 32) * 1024, "the Q operands lie where the waves' sums go at the end");
    const int per = a.T * (a.q_heads / a.kv_heads);
    const bool prompt = (int)blockIdx.x < a.prefix_blocks;
    if constexpr (NQP == NQO) {
        const Part p = prompt ? prompt_part(a, per, NQP * 16) : own_part(a, per, NQP * 16);
        part_rows<D, NQP>(a, p, os, ms, ls, bs);
    } else if (prompt) {
        part_rows<D, NQP>(a, prompt_part(a, per, NQP * 16), os, ms, ls, bs);
    } else {
        part_rows<D, NQO>(a, own_part(a, per, NQO * 16), os, ms, ls, bs);
    }
}

// Joins the parts: D / 4 threads a row, a thread four dims, kJoin parts' loads in flight.
constexpr int kJoin = 8;
template <int D>
__global__ void __launch_bounds__(256) shared_join(Kv4Shared a) {
    const int group = a.q_heads / a.kv_heads, per = a.T * group, d = threadIdx.x % (D / 4) * 4;
    const long long e = ((long long)blockIdx.x * 256 + threadIdx.x) / (D / 4);
    const int r = (int)(e % per), h = (int)(e / per % a.kv_heads);
    const long long i = e / ((long long)per * a.kv_heads);
    if (i >= a.n) return;
    const int j = a.group[i];
    const int end = j + 1 < a.groups ? a.gstart[j + 1] : a.n, start = a.gstart[j], prompt = a.glen[j] ? a.gsplits[j] : 0;
    const int first = a.first[i], own = (i + 1 < a.n ? a.first[i + 1] : a.own_splits) - first;
    const long long step = (long long)a.kv_heads * (end - start) * per, own_step = (long long)a.kv_heads * per;
    const long long p0 = a.gpart[j] + ((long long)h * (end - start) + (i - start)) * per + r;
    const long long o0 = a.own_part + ((long long)first * a.kv_heads + h) * per + r;
    const int parts = prompt + own;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, sum = 0.f;
    for (int s0 = 0; s0 < parts; s0 += kJoin) {
        f32x4 o[kJoin];
        float2 ml[kJoin];
#pragma unroll
        for (int s = 0; s < kJoin; ++s) {
            const int k = s0 + s;
            const float* p = a.part + (k < prompt ? p0 + k * step : o0 + (k - prompt) * own_step) * (D + 4);
            const bool in = k < parts;
            o[s] = in ? *(const f32x4*)(p + d) : f32x4{0.f, 0.f, 0.f, 0.f};
            ml[s] = in ? *(const float2*)(p + D) : make_float2(-INFINITY, 0.f);
        }
        float mn = m;
#pragma unroll
        for (int s = 0; s < kJoin; ++s) mn = fmaxf(mn, ml[s].x);
        const float mz = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - mz);
        x *= al;
        sum *= al;
        m = mn;
#pragma unroll
        for (int s = 0; s < kJoin; ++s) {
            const float f = __builtin_amdgcn_exp2f(ml[s].x - mz);
            sum += f * ml[s].y;
            x += f * o[s];
        }
    }
    const int t = r / group;
    Out(a, (long long)a.seq[i] * a.TT + t, h * group + r - t * group).template store<4>(a, (float*)&x, sum, d);
}

constexpr int kPromptSplits = 128, kOwnSplits = 128;
template <int D>
static hipError_t launch(Kv4Shared& a, hipStream_t st) {
    const int group = a.q_heads / a.kv_heads, per = a.T * group;
    const auto members = [&](int j) { return (j + 1 < a.groups ? a.gstart[j + 1] : a.n) - a.gstart[j]; };
    int most = 0;
    for (int j = 0; j < a.groups; ++j)
        if (a.glen[j]) most = std::max(most, members(j) * per);
    const int nqp = most > 16 ? 2 : 1, nqo = per > 16 ? 2 : 1;
    const auto row_tiles = [](int rows, int nq) { return (rows + nq * 16 - 1) / (nq * 16); };
    const auto own_tiles = [&](int i) { return ((a.pos[i] + a.T - 1) >> 5) + 1; };
    long long work = 0;                                  // tiles of all blocks
    for (int j = 0; j < a.groups; ++j)
        work += (long long)((a.glen[j] + 31) >> 5) * a.kv_heads * row_tiles(members(j) * per, nqp);
    for (int i = 0; i < a.n; ++i) work += (long long)own_tiles(i) * a.kv_heads * row_tiles(per, nqo);
    long long rows = 0, blocks = 0;
    for (int tiles = (int)std::max<long long>(8, (work + 511) / 512);; tiles *= 2) {
        rows = blocks = 0;
        bool least = true;
        for (int j = 0; j < a.groups; ++j) {
            const int len = (a.glen[j] + 31) >> 5, s = std::min(kPromptSplits, (len + tiles - 1) / tiles);
            least &= s <= 1;
            a.gfirst[j] = (int)blocks;
            a.gpart[j] = (int)rows;
            a.gsplits[j] = (uint16_t)std::max(1, s);
            blocks += (long long)s * a.kv_heads * row_tiles(members(j) * per, nqp);
            rows += (long long)s * a.kv_heads * members(j) * per;
        }
        a.prefix_blocks = (int)blocks;
        a.own_part = rows;
        int z = 0;
        for (int i = 0; i < a.n; ++i) {
            const int s = std::min(kOwnSplits, (own_tiles(i) + tiles - 1) / tiles);
            least &= s == 1;
            a.first[i] = (uint16_t)z;
            z += s;
        }
        a.own_splits = z;
        rows += (long long)z * a.kv_heads * per;
        blocks += (long long)z * a.kv_heads * row_tiles(per, nqo);
        if (rows <= kv4_shared_room(D)) break;
        if (least) return hipErrorInvalidValue;
    }
    for (int j = a.groups; j < kGroupArgs; ++j) a.gfirst[j] = INT_MAX;
    for (int i = a.n; i < kSeqArgs; ++i) a.first[i] = 0xffff;
    if (blocks > kLaunchBlocks) return hipErrorInvalidValue;
    const auto k = nqp == 1 ? shared_kernel<D, 1, 1> : nqo == 1 ? shared_kernel<D, 2, 1> : shared_kernel<D, 2, 2>;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, a);
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    const long long threads = (long long)a.n * a.kv_heads * per * (D / 4);
    hipLaunchKernelGGL(shared_join<D>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}
hipError_t launch_attn_kv4_shared(Kv4Shared& a, hipStream_t st) {
    return a.D == 256 ? launch<256>(a, st) : a.D == 128 ? launch<128>(a, st) : launch<64>(a, st);
}

}  // namespace q35
