// Log probabilities of given tokens (q35_logprobs.hip) and attention of answers that share prompts over the 4-bit
// cache (q35_kv4_shared.hip): what their entry points pass to the kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "q35_kv4.h"

struct q35_logprobs;

namespace q35 {

// Attention of answers that share prompts. The launch's sequences are sorted by prompt; entry j is the prompt of gcount
// sequences from gstart on (those without one are the last entry, of length 0). Each block leaves partial results.
constexpr int kEntryArgs = 64;       // prompts of one launch
struct Kv4Shared {
    const uint8_t *prefix, *cache;                       // layer bases
    size_t prefix_lane, prefix_region, lane_bytes, region;
    HeadView q, gate, out;                               // gate.p null: none; row i * TT + t is sequence i's
    int q_heads, kv_heads, D, T, TT;                     // T of a sequence's TT rows are this launch's
    float scale;
    float* part;
    int n, entries;
    int prompt_blocks, own_splits, own_units, own_part;  // (set by the launcher, as all below but pos, lane, seq, glen, glane, gstart)
    uint32_t per_inv, group_inv, kv_inv;                 // reciprocals of T x group, group and kv_heads
    alignas(16) int pos[kSeqArgs];
    alignas(16) uint16_t lane[kSeqArgs];
    alignas(16) uint16_t first[kSeqArgs];                // first split of each sequence's own slots; 0xffff past the last
    alignas(16) uint8_t seq[kSeqArgs];                   // its row block in the views
    alignas(16) int gfirst[kEntryArgs], gpart[kEntryArgs], glen[kEntryArgs], gtile[kEntryArgs];   // first block, first partial tile, slots, first tile to join
    alignas(16) uint16_t glane[kEntryArgs], gstart[kEntryArgs], gcount[kEntryArgs], gsplits[kEntryArgs];
};
static_assert(sizeof(Kv4Shared) <= 4096, "kernel arguments");
// Partial results lie in tiles of 16 rows: a launch needs at least kv_heads times kv4_tiles of each prompt's rows and of each
// sequence's (T x group), and has room for so many.
inline long long kv4_tiles(long long rows) { return (rows + 15) / 16; }
long long kv4_shared_room(int D);
hipError_t launch_attn_kv4_shared(Kv4Shared& a, hipStream_t st);

constexpr int kTopMost = 32;         // alternatives of a row
struct LogprobArgs {
    const void* logits;              // [rows][ld], f32 or bf16
    long long ld;
    int bf16, rows, vocab, top;
    double c;                        // log2(e) / temperature
    const int* targets;              // [rows]; null: none
    float *logprobs, *entropy, *top_logprobs;
    int *ranks, *top_ids;            // null where not wanted
    char* ws;                        // logprob_ws_bytes()
    int parts;                       // blocks of a row (set by the launcher)
};
size_t logprob_ws_bytes();
// A caller's wishes, looked over, but for logits, ld, dtype and the workspace.
LogprobArgs logprob_args(const q35_logprobs& d, int rows, int vocab);
hipError_t launch_logprobs(LogprobArgs a, hipStream_t st);

}  // namespace q35
