// Log probabilities of given tokens (q35_logprobs.hip) and attention of answers that share prompts over the 4-bit
// cache (q35_kv4_shared.hip): what their entry points pass to the kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "q35_kv4.h"

namespace q35 {

// Attention of answers that share prompts. The launch's sequences are sorted by prompt; group j's are gstart[j] ..
// gstart[j + 1] - 1 (those without a prompt the last group, of length 0). Each block leaves a partial result of its rows.
constexpr int kGroupArgs = 64;       // prompts of one launch
struct Kv4Shared {
    const uint8_t *prefix, *cache;                       // layer bases
    size_t prefix_lane, prefix_region, lane_bytes, region;
    HeadView q, gate, out;                               // gate.p null: none; row i * TT + t is sequence i's
    int q_heads, kv_heads, D, T, TT;                     // T of a sequence's TT rows are this launch's
    float scale;
    float* part;
    int n, groups;
    int prefix_blocks, own_splits;                       // (set by the launcher, as all below but pos, lane, seq, glen, glane, gstart)
    long long own_part;                                  // first partial row of the sequences' own slots
    alignas(16) int pos[kSeqArgs];
    alignas(16) uint16_t lane[kSeqArgs];
    alignas(16) uint16_t first[kSeqArgs];                // first split of each sequence's own slots; 0xffff past the last
    alignas(16) uint8_t seq[kSeqArgs], group[kSeqArgs];  // which row block of the views it is; its prompt
    alignas(16) int gfirst[kGroupArgs], gpart[kGroupArgs], glen[kGroupArgs];   // first block, first partial row, slots
    alignas(16) uint16_t glane[kGroupArgs], gstart[kGroupArgs], gsplits[kGroupArgs];
};
static_assert(sizeof(Kv4Shared) <= 4096, "kernel arguments");
// Partial rows that a launch of `rows` rows (sequences x T x query heads) needs at least, and has.
inline long long kv4_shared_need(long long rows) { return 2 * rows; }
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
hipError_t launch_logprobs(LogprobArgs a, hipStream_t st);

}  // namespace q35
