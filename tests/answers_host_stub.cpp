// The host half of q35_answers.cpp without a GPU, beside that of q35_kv4.cpp: its launches counted, and what the last one
// was given kept for the tests to look at.
#include "kv4_host_stub.cpp"

#include "q35_answers.h"

static q35::Kv4Shared g_shared;
static q35::AxisHeadArgs g_axes;
static long long g_rows, g_room;

namespace q35 {
hipError_t launch_heads(AxisHeadArgs& a, int n, hipStream_t) {
    g_axes = a;
    g_rows += (long long)n * a.T;
    return count();
}
hipError_t launch_logprobs(LogprobArgs, hipStream_t) { return count(); }
long long kv4_shared_room(int) { return g_room ? g_room : 2064; }
hipError_t launch_attn_kv4_shared(Kv4Shared& a, hipStream_t) {
    g_shared = a;
    g_rows += (long long)a.n * a.T;
    return count();
}
}  // namespace q35

extern "C" {
void stub_room(long long rows) { g_room = rows; }
long long stub_rows() { const long long r = g_rows; g_rows = 0; return r; }
int stub_axis(int pair) { return g_axes.axis_of[pair >> 4] >> 2 * (pair & 15) & 3; }
int stub_axes() { return g_axes.axes; }
// What the last launch of shared attention took: sequences, prompts, T; then per sequence its row block, prompt and position.
void stub_shared(int32_t* out) {
    *out++ = g_shared.n;
    *out++ = g_shared.entries;
    *out++ = g_shared.T;
    for (int i = 0; i < g_shared.n; ++i) {
        int j = 0;
        while (j + 1 < g_shared.entries && g_shared.gstart[j + 1] <= i) ++j;
        *out++ = g_shared.seq[i];
        *out++ = g_shared.glen[j] ? g_shared.glane[j] : -1;
        *out++ = g_shared.glen[j];
        *out++ = g_shared.pos[i];
    }
}
}
