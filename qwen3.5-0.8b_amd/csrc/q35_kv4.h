// A K/V cache in 4 bits, the kernels around it, and its layout (q35_kv4.hip).
//
// A head's row of D dims (64, 128 or 256) at one slot is held in groups of 32 consecutive dims.
// A group has one scale byte b, standing for 2^(b - 127) -- the smallest power of two whose
// largest code covers the group's largest magnitude -- and 32 codes of 4 bits: sign, 2 exponent bits
// and 1 mantissa bit, the values +- (0, 0.5, 1, 1.5, 2, 3, 4, 6), which is what gfx950's
// v_cvt_scalef32_pk_bf16_fp4 turns into bf16 (exactly: a code has 2 significant bits), two
// values an instruction, scale included. b = 255 marks a group that held an infinity or a NaN;
// the instruction gives NaN for it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace q35 {

// Layout. A (layer, lane, kv head) region is a run of 32-slot tiles of 34 D bytes:
//   [K codes 16 D][V codes 16 D][K scales D][V scales D]
// Codes lie in the order in which a wave's lanes want them for the 16x16x32 MFMAs: each lane
// (m = lane % 16, g = lane / 16) owns D/4 bytes of the K and of the V codes, stored as D/64 pieces of
// 1 KiB that hold 16 bytes of every lane, so that every load instruction reads 1 KiB in a row.
//   K (A operand of S^T = K Q^T, 2 halves of 16 slots): lane (m, g) holds dims [g D/4, (g+1) D/4)
//     of slots m and 16 + m; MFMA step s takes dims g D/4 + 8 s + (0..7), one dword.
//   V (A operand of O^T = V^T P^T, k = the tile's 32 slots): lane (m, g) holds dims
//     [m D/16, (m+1) D/16) of the 8 slots 4g + (0..3), 16 + 4g + (0..3) -- the slots whose
//     probabilities S^T's accumulators leave in lanes (., g), so P needs no move between lanes.
__host__ __device__ inline size_t kv4_tile_bytes(int D) { return (size_t)34 * D; }
__host__ __device__ inline size_t kv4_region_bytes(int D, int cap) { return (size_t)((cap + 31) / 32) * kv4_tile_bytes(D); }
// Byte of the pair of codes (d, d + 1), d even, of a tile's slot tk (0 .. 31).
__host__ __device__ inline int kv4_k_code(int D, int tk, int d) {
    const int lane = d / (D / 4) * 16 + tk % 16, off = tk / 16 * (D / 8) + d % (D / 4) / 2;
    return off / 16 * 1024 + lane * 16 + off % 16;
}
__host__ __device__ inline int kv4_v_code(int D, int tk, int d) {
    const int g = tk % 16 / 4, jj = tk / 16 * 4 + tk % 4;
    const int lane = g * 16 + d / (D / 16), off = jj * (D / 32) + d % (D / 16) / 2;
    return 16 * D + off / 16 * 1024 + lane * 16 + off % 16;
}
// Scale byte of the group of dims [32 blk, 32 blk + 32): K's are the bytes of a lane's blob (2 or 4
// bytes a lane; at D = 64 two lane groups share a group of dims), V's the 8 slots of a lane group.
__host__ __device__ inline int kv4_k_scale(int D, int tk, int blk) {
    const int per = D >= 256 ? 2 : 1;
    return 32 * D + (blk / per * 16 + tk % 16) * 2 * per + tk / 16 * per + blk % per;
}
__host__ __device__ inline int kv4_v_scale(int D, int tk, int blk) {
    return 33 * D + blk * 32 + tk % 16 / 4 * 8 + tk / 16 * 4 + tk % 4;
}

// Rows of heads in a caller's buffer: element (row r, head h, dim d) at p[r * row + h * head + d].
struct HeadView { const uint16_t* p; long long row, head; };

constexpr int kSeqArgs = 256;        // sequences of one launch (their positions travel as kernel arguments)
constexpr int kLaunchBlocks = (1 << 24) - 1;   // blocks of 256 threads of one launch: HIP counts its threads in 32 bits
struct HeadArgs {
    HeadView q, k, v, q_out, k_out, v_out;   // v, q_out, k_out, v_out: p null where not wanted
    const uint16_t *q_norm, *k_norm;
    int q_heads, kv_heads, D, rot, T;
    double eps, rate;            // rate: -2 log2(theta) / rot, the angles' exponents' step
    uint8_t* cache;              // layer base, or null
    size_t lane_bytes, region;   // bytes of a lane (its kv_heads regions), of a region
    uint32_t q_inv, kv_inv;      // 2^32 / heads + 1 (set by the launcher)
    int pos[kSeqArgs];
    uint16_t lane[kSeqArgs];
};
// q and k: RMS norm per head and rotation; with a.cache, k and v through 4 bits into the cache. n <= kSeqArgs
// sequences of T rows, n T <= kHeadRows.
constexpr int kHeadRows = 4 * kLaunchBlocks;   // (a block takes four of many rows)
hipError_t launch_heads(HeadArgs& a, int n, hipStream_t st);

struct Kv4Attn {
    const uint8_t* cache;        // layer base
    size_t lane_bytes, region;
    HeadView q, gate, out;       // gate.p null: none
    int q_heads, kv_heads, D, T;
    int window, sinks;           // window 0: every slot up to the row's own
    float scale;
    float* part;                 // split workspace (kv4_part_floats())
    int n, splits;               // sequences and their splits together (the launcher sets these and first)
    alignas(16) int pos[kSeqArgs];
    alignas(16) uint16_t lane[kSeqArgs];
    alignas(16) uint16_t first[kSeqArgs];   // first split of each sequence; 0xffff past the last
};
// Blocks of an unsplit sequence: for each kv head one for every 32 rows (T times its query heads), or for 16 rows or fewer.
inline int kv4_attn_items(int q_heads, int kv_heads, int T) {
    const long long rows = (long long)T * (q_heads / kv_heads), of = rows > 16 ? 32 : 16;
    return (int)(kv_heads * ((rows + of - 1) / of));
}
size_t kv4_part_floats();
hipError_t launch_attn_kv4(Kv4Attn& a, int n, hipStream_t st);

// Row-major rows <-> the cache, n_slots from slot0 of lanes lane0 .. lane0 + n_lanes: codes
// [n_lanes][kv_heads][n_slots][D/2], scales [..][D/32].
struct Kv4Copy {
    uint8_t* cache;
    size_t lane_bytes, region;
    int kv_heads, D, lane0, n_lanes, slot0, n_slots;
    uint8_t *kc, *ks, *vc, *vs;
};
hipError_t launch_kv4_copy(const Kv4Copy& a, bool write, hipStream_t st);

// Verification of drafts (q35_verify.hip).
struct VerifyScale { double c, low; };   // log2(e) / temperature; -1100 / c
struct VerifyArgs {
    const void *logits, *draft_logits;   // [n][k + 1][ld], [n][k][ldd] (null: drafts are certain); f32 or bf16
    long long ld, ldd;
    int bf16, n, k, vocab;
    double inv_temp;                     // 0: greedy
    VerifyScale scale;
    const int* drafts;                   // [n][k]; the first negative one ends a lane's drafts
    const float* u;                      // [n][k + 1]
    int *accepted, *tokens;              // [n], [n][k + 1]
    double* stats;                       // workspace
    int chunks, chunk;                   // a row's chunks and their elements (set by the launcher)
    void set_temperature(double t) {
        inv_temp = t == 0.0 ? 0.0 : 1.0 / t;
        scale.c = inv_temp * 1.4426950408889634074;
        scale.low = t == 0.0 ? 0.0 : -1100.0 / scale.c;
    }
};
inline bool verify_temperature_ok(double t) { return t == 0.0 || (t >= 1e-3 && t <= 1e300); }
constexpr int kVerifyDrafts = 8;
size_t verify_ws_doubles(int max_rows);
hipError_t launch_verify(VerifyArgs& a, hipStream_t st);

}  // namespace q35
