// C ABI of heads at positions on several axes, attention of answers that share prompts, and token log
// probabilities (include/q35.h): argument checks and launches. Calls are enqueued on the engine's stream.
#include <hip/hip_runtime.h>

#include "q35_answers.h"
#include "q35_kv4_host.h"

using namespace q35;

// The axes' positions and the pairs' axes, two bits each.
static AxisHeadArgs axis_args(const HeadArgs& h, const q35_positions& at, const uint8_t* axis) {
    AxisHeadArgs a{};
    static_cast<HeadArgs&>(a) = h;
    if (!h.rot) return a;
    REQ(at.pos && axis, Q35_ERR_ARG, "null positions or axes");
    REQ((uintptr_t)at.pos % 4 == 0, Q35_ERR_ARG, "misaligned positions");
    REQ(at.row_stride >= 0 && at.axis_stride >= 0, Q35_ERR_ARG, "positions: negative stride");
    a.axis_pos = at.pos;
    a.row_step = at.row_stride;
    bool named[kAxes] = {};
    for (int i = 0; i < h.rot / 2; ++i) {
        REQ(axis[i] < kAxes, Q35_ERR_ARG, "a pair's axis is 0 .. 3");
        named[axis[i]] = true;
        a.axes = std::max(a.axes, axis[i] + 1);
        a.axis_of[i >> 4] |= (uint32_t)axis[i] << 2 * (i & 15);
    }
    for (int x = 0; x < a.axes; ++x) a.axis_at[x] = (named[x] ? x : a.axes - 1) * at.axis_stride;
    return a;
}

LogprobArgs q35::logprob_args(const q35_logprobs& d, int rows, int vocab) {
    REQ(rows > 0, Q35_ERR_ARG, "bad row count");
    REQ(vocab >= 1 && vocab <= 1 << 20, Q35_ERR_ARG, "vocab is 1 .. 1048576");
    REQ(d.temperature >= 1e-3 && d.temperature <= 1e3, Q35_ERR_ARG, "temperature is 0.001 .. 1000");
    REQ(d.top >= 0 && d.top <= std::min(kTopMost, vocab), Q35_ERR_ARG, "top is 0 .. 32, at most vocab");
    REQ(d.targets || (!d.logprobs && !d.ranks), Q35_ERR_ARG, "log probabilities and ranks need targets");
    LogprobArgs a{};
    a.rows = rows; a.vocab = vocab;
    a.top = d.top_ids || d.top_logprobs ? d.top : 0;
    a.c = 1.4426950408889634074 / d.temperature;
    a.targets = d.targets; a.logprobs = d.logprobs; a.ranks = d.ranks; a.entropy = d.entropy;
    a.top_ids = d.top_ids; a.top_logprobs = d.top_logprobs;
    return a;
}

extern "C" {

int q35_op_qk_norm_rope_axes(q35_engine* e, const q35_heads* h, int kv_heads, int head_dim, const q35_positions* at,
                             const uint8_t* axis, int rows) {
    return guard([&] {
        REQ(e && h && at, Q35_ERR_ARG, "null argument");
        const AxisHeadArgs a = axis_args(head_args(*h, kv_heads, head_dim, 1, rows, false), *at, axis);
        const EngineView ev = engine_view(e);
        OnDevice on(ev.device);
        const int32_t zero = 0;
        run_heads(a, nullptr, &zero, 1, ev.st);
    });
}

int q35_op_kv4_append_axes(q35_engine* e, q35_kv4* c, int layer, const int32_t* lanes, const int32_t* slots, int n, int T,
                           const q35_heads* h, const q35_positions* at, const uint8_t* axis) {
    return guard([&] {
        check_cache(e, c);
        REQ(h && at, Q35_ERR_ARG, "null argument");
        check_seqs(c, layer, lanes, slots, n, T, true);
        AxisHeadArgs a = axis_args(head_args(*h, c->kv_heads, c->D, n, T, true), *at, axis);
        a.cache = c->mem + layer * c->layer_bytes();
        a.lane_bytes = c->lane_bytes(); a.region = c->region();
        const EngineView ev = engine_view(e);
        OnDevice on(ev.device);
        run_heads(a, lanes, slots, n, ev.st);
        for (int i = 0; i < n; ++i) c->held(layer, lanes ? lanes[i] : i) = slots[i] + T;
    });
}

int q35_op_attn_kv4_shared(q35_engine* e, q35_kv4* prefix, q35_kv4* c, int layer, const int32_t* prefix_lanes,
                           const int32_t* prefix_lens, const int32_t* lanes, const int32_t* pos, int n, int T, int q_heads,
                           const q35_view* q, const q35_view* gate, float scale, const q35_view* out) {
    return guard([&] {
        check_cache(e, prefix);
        check_cache(e, c);
        REQ(prefix_lanes && prefix_lens && q && out, Q35_ERR_ARG, "null argument");
        REQ(prefix->kv_heads == c->kv_heads && prefix->D == c->D, Q35_ERR_ARG, "the caches' heads differ");
        REQ(layer < prefix->layers, Q35_ERR_ARG, "layer out of range");
        check_seqs(c, layer, lanes, pos, n, T, false);
        const auto has = [&](int i) { return prefix_lanes[i] >= 0 && prefix_lens[i] != 0; };
        for (int i = 0; i < n; ++i) {
            REQ(prefix_lens[i] >= 0, Q35_ERR_ARG, "negative prefix length");
            if (!has(i)) continue;
            REQ(prefix_lanes[i] < prefix->lanes, Q35_ERR_ARG, "prefix lane out of range");
            REQ(prefix_lens[i] <= prefix->held(layer, prefix_lanes[i]), Q35_ERR_STATE, "prefix slots that the lane does not hold");
            REQ(prefix != c || prefix_lanes[i] != (lanes ? lanes[i] : i), Q35_ERR_ARG, "a lane cannot be its own prefix");
        }
        REQ(q_heads > 0 && q_heads <= 1024 && q_heads % c->kv_heads == 0, Q35_ERR_ARG,
            "q_heads must be a multiple of the cache's kv_heads");
        REQ(std::isfinite(scale * 1.44269504f), Q35_ERR_ARG, "scale must be finite, times log2(e) too");
        Kv4Shared a{};
        const HeadView qv = view(*q, "q"), ov = view(*out, "out"), gv = gate ? maybe_view(*gate, "gate") : HeadView{nullptr, 0, 0};
        check_out(ov, q_heads, n * T, c->D, "out");
        const EngineView ev = engine_view(e);
        a.prefix = prefix->mem + layer * prefix->layer_bytes();
        a.prefix_lane = prefix->lane_bytes(); a.prefix_region = prefix->region();
        a.cache = c->mem + layer * c->layer_bytes();
        a.lane_bytes = c->lane_bytes(); a.region = c->region();
        a.q_heads = q_heads; a.kv_heads = c->kv_heads; a.D = c->D; a.TT = T; a.scale = scale; a.part = ev.kv4_part;
        OnDevice on(ev.device);
        // A launch takes sequences out of kSeqArgs neighbours, as many of their rows as the partial results have room for.
        const long long room = kv4_shared_room(c->D) / c->kv_heads;
        const int group = q_heads / c->kv_heads, rows = (int)std::min<long long>({T, std::max(room / 2 * 16 / group, 1LL), 32768 / group});
        std::vector<int> order;
        for (int i0 = 0; i0 < n; i0 += kSeqArgs) {
            order.resize(std::min(kSeqArgs, n - i0));
            for (int i = 0; i < (int)order.size(); ++i) order[i] = i0 + i;
            const auto less = [&](int x, int y) {        // by prompt, those without one last
                if (!has(x) || !has(y)) return has(x) && !has(y);
                return prefix_lanes[x] != prefix_lanes[y] ? prefix_lanes[x] < prefix_lanes[y] : prefix_lens[x] < prefix_lens[y];
            };
            std::stable_sort(order.begin(), order.end(), less);
            for (int t0 = 0; t0 < T; t0 += rows) {
                a.T = std::min(rows, T - t0);
                const auto moved = [&](HeadView v) { return HeadView{v.p ? v.p + ((long long)i0 * T + t0) * v.row : nullptr, v.row, v.head}; };
                a.q = moved(qv); a.gate = moved(gv); a.out = moved(ov);
                for (size_t k = 0; k < order.size();) {
                    a.n = a.entries = 0;
                    long long used = 0;
                    for (; k < order.size(); ++k) {
                        const int i = order[k], next = a.n == 0 || less(order[k - 1], i), per = a.T * group;
                        const long long with = next ? 0 : a.n - a.gstart[a.entries - 1];
                        const long long more = kv4_tiles(per) + kv4_tiles((with + 1) * per) - kv4_tiles(with * per);
                        if (a.n && (a.entries + next > kEntryArgs || used + more > room)) break;
                        used += more;
                        if (next) {
                            a.gstart[a.entries] = (uint16_t)a.n;
                            a.glane[a.entries] = (uint16_t)(has(i) ? prefix_lanes[i] : 0);
                            a.glen[a.entries++] = has(i) ? prefix_lens[i] : 0;
                        }
                        a.pos[a.n] = pos[i] + t0;
                        a.lane[a.n] = (uint16_t)(lanes ? lanes[i] : i);
                        a.seq[a.n++] = (uint8_t)(i - i0);
                    }
                    HCK(launch_attn_kv4_shared(a, ev.st));
                }
            }
        }
    });
}

int q35_op_token_logprobs(q35_engine* e, const q35_logprobs* d, int rows, int vocab) {
    return guard([&] {
        REQ(e && d && d->logits, Q35_ERR_ARG, "null argument");
        LogprobArgs a = logprob_args(*d, rows, vocab);
        REQ(d->ld >= vocab, Q35_ERR_ARG, "row stride below vocab");
        REQ(d->dtype == 0 || d->dtype == 1, Q35_ERR_ARG, "dtype is 0 (float32) or 1 (bfloat16)");
        REQ((uintptr_t)d->logits % (d->dtype ? 2 : 4) == 0, Q35_ERR_ARG, "misaligned logits");
        a.logits = d->logits; a.ld = d->ld; a.bf16 = d->dtype;
        const EngineView ev = engine_view(e);
        a.ws = ev.logprob_ws;
        OnDevice on(ev.device);
        HCK(launch_logprobs(a, ev.st));
    });
}

}  // extern "C"
