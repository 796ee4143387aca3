// C ABI of the 4-bit K/V cache, the operators around it and the sampled draft verification
// (include/q35.h): argument checks and launches. Calls are enqueued on the engine's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <vector>

#include "q35_host.h"
#include "q35_kv4.h"

using namespace q35;

struct q35_kv4 {
    q35_engine* eng = nullptr;
    int device = 0, layers = 0, lanes = 0, cap = 0, kv_heads = 0, D = 0;
    uint8_t* mem = nullptr;          // [layers][lanes][kv_heads] regions
    std::vector<int> len;            // [layers][lanes] slots held
    size_t region() const { return kv4_region_bytes(D, cap); }
    size_t lane_bytes() const { return (size_t)kv_heads * region(); }
    size_t layer_bytes() const { return (size_t)lanes * lane_bytes(); }
    int& held(int layer, int lane) { return len[(size_t)layer * lanes + lane]; }
};

namespace {

// The engine's device as the calling thread's current one, for as long as the call lasts.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        int now = 0;
        HCK(hipGetDevice(&now));
        if (now != device) {
            HCK(hipSetDevice(device));
            before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

void check_dim(int D) { REQ(D == 64 || D == 128 || D == 256, Q35_ERR_ARG, "head_dim is 64, 128 or 256"); }

// A view of rows: 16-byte loads and stores from every (row, head).
HeadView view(const q35_view& v, const char* what) {
    const auto bad = [&](const char* why) { return Q35Error(Q35_ERR_ARG, std::string(what) + ": " + why); };
    if (!v.ptr) throw bad("null pointer");
    if ((uintptr_t)v.ptr % 16 || v.row_stride % 8 || v.head_stride % 8)
        throw bad("the pointer must be 16-byte aligned and the strides multiples of 8 elements");
    if (v.row_stride < 0 || v.head_stride < 0) throw bad("negative stride");
    return {v.ptr, v.row_stride, v.head_stride};
}
HeadView maybe_view(const q35_view& v, const char* what) { return v.ptr ? view(v, what) : HeadView{nullptr, 0, 0}; }
// An output's heads and rows must not share elements.
void check_out(const HeadView& v, int heads, int rows, int D, const char* what) {
    if (!v.p) return;
    const bool apart = (heads == 1 || v.head >= D) && (rows == 1 || v.row >= D) &&
                       (heads == 1 || rows == 1 || v.row >= (heads - 1) * v.head + D || v.head >= (rows - 1) * v.row + D);
    REQ(apart, Q35_ERR_ARG, std::string(what) + ": rows or heads overlap");
}

// Sequences of a call on cache c's `layer`: lanes in range (i when null); each position at most the lane's
// length for an append (which then holds pos + T slots), pos + T at most the length for a read.
void check_seqs(q35_kv4* c, int layer, const int32_t* lanes, const int32_t* pos, int n, int T, bool append) {
    REQ(layer >= 0 && layer < c->layers, Q35_ERR_ARG, "layer out of range");
    REQ(n > 0 && T > 0 && pos, Q35_ERR_ARG, "bad sequence count, row count or positions");
    REQ((long long)n * T <= INT32_MAX, Q35_ERR_ARG, "bad sequence or row count");
    std::vector<char> seen(append ? c->lanes : 0, 0);
    for (int i = 0; i < n; ++i) {
        const int l = lanes ? lanes[i] : i;
        REQ(l >= 0 && l < c->lanes, Q35_ERR_ARG, "lane out of range");
        REQ(pos[i] >= 0 && T <= c->cap && pos[i] <= c->cap - T, Q35_ERR_CAP, "rows past the cache's capacity");
        if (append) {
            REQ(!seen[l], Q35_ERR_ARG, "a lane occurs twice in one append");
            seen[l] = 1;
            REQ(pos[i] <= c->held(layer, l), Q35_ERR_STATE, "append behind the lane's last slot would leave a gap");
        } else {
            REQ(pos[i] <= c->held(layer, l) - T, Q35_ERR_STATE, "rows at slots that the lane does not hold yet");
        }
    }
}

void check_cache(q35_engine* e, q35_kv4* c) {
    REQ(e && c, Q35_ERR_ARG, "null argument");
    REQ(c->eng == e, Q35_ERR_ARG, "the cache belongs to another engine");
}

HeadArgs head_args(const q35_heads& s, int kv_heads, int D, int n, int T, bool cached) {
    check_dim(D);
    REQ(kv_heads > 0 && kv_heads <= 1024 && s.q_heads >= 0 && s.q_heads <= 1024, Q35_ERR_ARG, "head count out of range");
    REQ(s.rot_dim >= 0 && s.rot_dim <= D && s.rot_dim % 2 == 0, Q35_ERR_ARG, "rot_dim is even and at most head_dim");
    REQ(s.rot_dim == 0 || (s.theta > 0.0 && std::isfinite(s.theta)), Q35_ERR_ARG, "theta must be positive");
    REQ(s.eps >= 0.0 && std::isfinite(s.eps), Q35_ERR_ARG, "eps must not be negative");
    REQ(n > 0 && T > 0 && T <= kHeadRows && (long long)n * T <= INT32_MAX, Q35_ERR_ARG, "bad sequence or row count");
    REQ((s.q.ptr != nullptr) == (s.q_out.ptr != nullptr), Q35_ERR_ARG, "q and q_out go together");
    REQ(!s.q.ptr || s.q_heads > 0, Q35_ERR_ARG, "q without q_heads");
    REQ((!s.q.ptr || s.q_norm) && s.k_norm, Q35_ERR_ARG, "null norm weight");
    REQ((uintptr_t)s.q_norm % 8 == 0 && (uintptr_t)s.k_norm % 8 == 0, Q35_ERR_ARG, "norm weights must be 8-byte aligned");
    HeadArgs a{};
    a.q = maybe_view(s.q, "q");
    a.k = view(s.k, "k");
    a.q_out = maybe_view(s.q_out, "q_out");
    if (cached) {
        a.v = view(s.v, "v");
        a.k_out = maybe_view(s.k_out, "k_out");
        a.v_out = maybe_view(s.v_out, "v_out");
    } else {
        REQ(!s.v.ptr && !s.v_out.ptr, Q35_ERR_ARG, "v has no norm or rotation");
        a.k_out = view(s.k_out, "k_out");
    }
    check_out(a.q_out, s.q_heads, n * T, D, "q_out");
    check_out(a.k_out, kv_heads, n * T, D, "k_out");
    check_out(a.v_out, kv_heads, n * T, D, "v_out");
    a.q_norm = s.q_norm; a.k_norm = s.k_norm;
    a.q_heads = s.q_heads; a.kv_heads = kv_heads; a.D = D; a.rot = s.rot_dim; a.T = T;
    a.eps = s.eps;
    a.rate = s.rot_dim ? -2.0 * std::log2(s.theta) / s.rot_dim : 0.0;
    return a;
}

// The launches of a call: at most kSeqArgs sequences and kHeadRows rows each.
void run_heads(HeadArgs a, const int32_t* lanes, const int32_t* pos, int n, hipStream_t st) {
    const auto move = [](HeadView& v, long long rows) { if (v.p) v.p += rows * v.row; };
    const int most = std::min(kSeqArgs, kHeadRows / a.T);
    for (int i0 = 0, m; i0 < n; i0 += m) {
        m = std::min(most, n - i0);
        for (int i = 0; i < m; ++i) {
            a.pos[i] = pos[i0 + i];
            a.lane[i] = (uint16_t)(lanes ? lanes[i0 + i] : i0 + i);
        }
        HCK(launch_heads(a, m, st));
        for (HeadView* v : {&a.q, &a.k, &a.v, &a.q_out, &a.k_out, &a.v_out}) move(*v, (long long)m * a.T);
    }
}

}  // namespace

extern "C" {

int q35_kv4_alloc(q35_engine* e, int layers, int lanes, int cap, int kv_heads, int head_dim, q35_kv4** out) {
    return guard([&] {
        REQ(e && out, Q35_ERR_ARG, "null argument");
        const EngineView ev = engine_view(e);
        check_dim(head_dim);
        REQ(layers > 0 && layers <= 1024 && lanes > 0 && lanes <= 65535 && kv_heads > 0 && kv_heads <= 1024 && cap > 0,
            Q35_ERR_ARG, "bad cache shape");
        REQ(cap <= ev.max_ctx, Q35_ERR_CAP, "cap exceeds engine max_ctx");
        OnDevice on(ev.device);
        std::unique_ptr<q35_kv4> c(new q35_kv4());
        c->eng = e; c->device = ev.device; c->layers = layers; c->lanes = lanes; c->cap = cap; c->kv_heads = kv_heads; c->D = head_dim;
        c->len.assign((size_t)layers * lanes, 0);
        const size_t bytes = (size_t)layers * c->layer_bytes();
        HCK(hipMalloc((void**)&c->mem, bytes));
        hipError_t rc = hipMemsetAsync(c->mem, 0, bytes, ev.st);
        if (rc == hipSuccess) rc = hipStreamSynchronize(ev.st);
        if (rc != hipSuccess) {
            (void)hipFree(c->mem);
            HCK(rc);
        }
        *out = c.release();
    });
}

int q35_kv4_free(q35_engine* e, q35_kv4* c) {
    return guard([&] {
        if (!c) return;
        OnDevice on(c->device);
        if (e) {
            check_cache(e, c);
            HCK(hipStreamSynchronize(engine_view(e).st));
        }
        HCK(hipFree(c->mem));
        delete c;
    });
}

int q35_kv4_set_len(q35_engine* e, q35_kv4* c, const int32_t* lanes, const int32_t* len, int n) {
    return guard([&] {
        check_cache(e, c);
        REQ(len && n > 0, Q35_ERR_ARG, "null argument");
        for (int i = 0; i < n; ++i) {
            const int l = lanes ? lanes[i] : i;
            REQ(l >= 0 && l < c->lanes, Q35_ERR_ARG, "lane out of range");
            REQ(len[i] >= 0 && len[i] <= c->cap, Q35_ERR_CAP, "length exceeds the cache's capacity");
        }
        for (int i = 0; i < n; ++i)
            for (int y = 0; y < c->layers; ++y) c->held(y, lanes ? lanes[i] : i) = len[i];
    });
}

int q35_kv4_len(q35_engine* e, q35_kv4* c, int layer, int lane, int32_t* out) {
    return guard([&] {
        check_cache(e, c);
        REQ(out, Q35_ERR_ARG, "null argument");
        REQ(layer >= 0 && layer < c->layers && lane >= 0 && lane < c->lanes, Q35_ERR_ARG, "layer or lane out of range");
        *out = c->held(layer, lane);
    });
}

static void kv4_copy(q35_engine* e, q35_kv4* c, int layer, int lane0, int n_lanes, int slot0, int n_slots, uint8_t* kc,
                     uint8_t* ks, uint8_t* vc, uint8_t* vs, bool write) {
    check_cache(e, c);
    REQ(kc && ks && vc && vs, Q35_ERR_ARG, "null argument");
    REQ(layer >= 0 && layer < c->layers, Q35_ERR_ARG, "layer out of range");
    REQ(lane0 >= 0 && n_lanes > 0 && n_lanes <= c->lanes && lane0 <= c->lanes - n_lanes, Q35_ERR_ARG, "lane out of range");
    REQ(slot0 >= 0 && n_slots > 0 && n_slots <= c->cap && slot0 <= c->cap - n_slots, Q35_ERR_CAP,
        "rows past the cache's capacity");
    for (int i = 0; i < n_lanes; ++i) {
        const int held = c->held(layer, lane0 + i);
        if (write) REQ(slot0 <= held, Q35_ERR_STATE, "write behind the lane's last slot would leave a gap");
        else REQ(slot0 <= held - n_slots, Q35_ERR_STATE, "rows at slots that the lane does not hold yet");
    }
    const EngineView ev = engine_view(e);
    OnDevice on(ev.device);
    Kv4Copy a{};
    a.cache = c->mem + layer * c->layer_bytes();
    a.lane_bytes = c->lane_bytes(); a.region = c->region();
    a.kv_heads = c->kv_heads; a.D = c->D; a.lane0 = lane0; a.n_lanes = n_lanes; a.slot0 = slot0; a.n_slots = n_slots;
    a.kc = kc; a.ks = ks; a.vc = vc; a.vs = vs;
    HCK(launch_kv4_copy(a, write, ev.st));
    if (write)
        for (int i = 0; i < n_lanes; ++i) {
            int& held = c->held(layer, lane0 + i);
            held = std::max(held, slot0 + n_slots);
        }
}

int q35_kv4_write(q35_engine* e, q35_kv4* c, int layer, int lane0, int n_lanes, int slot0, int n_slots,
                  const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales) {
    return guard([&] {
        kv4_copy(e, c, layer, lane0, n_lanes, slot0, n_slots, const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(k_scales),
                 const_cast<uint8_t*>(v_codes), const_cast<uint8_t*>(v_scales), true);
    });
}

int q35_kv4_read(q35_engine* e, q35_kv4* c, int layer, int lane0, int n_lanes, int slot0, int n_slots, uint8_t* k_codes,
                 uint8_t* k_scales, uint8_t* v_codes, uint8_t* v_scales) {
    return guard([&] {
        kv4_copy(e, c, layer, lane0, n_lanes, slot0, n_slots, k_codes, k_scales, v_codes, v_scales, false);
    });
}

int q35_op_qk_norm_rope(q35_engine* e, const q35_heads* h, int kv_heads, int head_dim, const int32_t* pos, int n, int T) {
    return guard([&] {
        REQ(e && h && pos, Q35_ERR_ARG, "null argument");
        const HeadArgs a = head_args(*h, kv_heads, head_dim, n, T, false);
        for (int i = 0; i < n; ++i)
            REQ(pos[i] >= 0 && pos[i] <= INT32_MAX - T, Q35_ERR_ARG, "position out of range");
        const EngineView ev = engine_view(e);
        OnDevice on(ev.device);
        run_heads(a, nullptr, pos, n, ev.st);
    });
}

int q35_op_kv4_append(q35_engine* e, q35_kv4* c, int layer, const int32_t* lanes, const int32_t* pos, int n, int T,
                      const q35_heads* h) {
    return guard([&] {
        check_cache(e, c);
        REQ(h, Q35_ERR_ARG, "null argument");
        check_seqs(c, layer, lanes, pos, n, T, true);
        HeadArgs a = head_args(*h, c->kv_heads, c->D, n, T, true);
        a.cache = c->mem + layer * c->layer_bytes();
        a.lane_bytes = c->lane_bytes(); a.region = c->region();
        const EngineView ev = engine_view(e);
        OnDevice on(ev.device);
        run_heads(a, lanes, pos, n, ev.st);
        for (int i = 0; i < n; ++i) c->held(layer, lanes ? lanes[i] : i) = pos[i] + T;
    });
}

int q35_op_attn_kv4(q35_engine* e, q35_kv4* c, int layer, const int32_t* lanes, const int32_t* pos, int n, int T,
                    int q_heads, const q35_view* q, const q35_view* gate, float scale, int window, int sinks,
                    const q35_view* out) {
    return guard([&] {
        check_cache(e, c);
        REQ(q && out, Q35_ERR_ARG, "null argument");
        check_seqs(c, layer, lanes, pos, n, T, false);
        REQ(q_heads > 0 && q_heads <= 1024 && q_heads % c->kv_heads == 0, Q35_ERR_ARG,
            "q_heads must be a multiple of the cache's kv_heads");
        REQ(window >= 0 && sinks >= 0, Q35_ERR_ARG, "window and sinks must not be negative");
        REQ(window > 0 || sinks == 0, Q35_ERR_ARG, "sinks go with a window");
        REQ(std::isfinite(scale * 1.44269504f), Q35_ERR_ARG, "scale must be finite, times log2(e) too");
        Kv4Attn a{};
        a.q = view(*q, "q");
        a.out = view(*out, "out");
        if (gate) a.gate = maybe_view(*gate, "gate");
        check_out(a.out, q_heads, n * T, c->D, "out");
        const EngineView ev = engine_view(e);
        a.cache = c->mem + layer * c->layer_bytes();
        a.lane_bytes = c->lane_bytes(); a.region = c->region();
        a.q_heads = q_heads; a.kv_heads = c->kv_heads; a.D = c->D; a.T = T;
        a.window = window; a.sinks = sinks; a.scale = scale; a.part = ev.kv4_part;
        OnDevice on(ev.device);
        const int most = std::min(kSeqArgs, kLaunchBlocks / kv4_attn_items(q_heads, c->kv_heads, T));
        for (int i0 = 0, m; i0 < n; i0 += m) {
            m = std::min(most, n - i0);
            for (int i = 0; i < m; ++i) {
                a.pos[i] = pos[i0 + i];
                a.lane[i] = (uint16_t)(lanes ? lanes[i0 + i] : i0 + i);
            }
            HCK(launch_attn_kv4(a, m, ev.st));
            for (HeadView* v : {&a.q, &a.gate, &a.out})
                if (v->p) v->p += (long long)m * T * v->row;
        }
    });
}

int q35_op_draft_verify(q35_engine* e, const q35_drafts* d, int n, int k, int vocab, int32_t* accepted, int32_t* tokens) {
    return guard([&] {
        REQ(e && d && accepted && tokens && d->logits && d->drafts && d->u, Q35_ERR_ARG, "null argument");
        const EngineView ev = engine_view(e);
        REQ(k >= 1 && k <= kVerifyDrafts, Q35_ERR_ARG, "drafts per lane are 1 .. 8");
        REQ(n > 0 && (long long)n * (k + 1) <= ev.max_rows, Q35_ERR_CAP, "rows exceed max_rows");
        REQ(vocab >= 1 && vocab <= 1 << 20, Q35_ERR_ARG, "vocab is 1 .. 1048576");
        REQ(d->ld >= vocab && (!d->draft_logits || d->draft_ld >= vocab), Q35_ERR_ARG, "row stride below vocab");
        REQ(d->dtype == 0 || d->dtype == 1, Q35_ERR_ARG, "dtype is 0 (float32) or 1 (bfloat16)");
        const uintptr_t el = d->dtype ? 2 : 4;
        REQ((uintptr_t)d->logits % el == 0 && (uintptr_t)d->draft_logits % el == 0, Q35_ERR_ARG, "misaligned logits");
        REQ(verify_temperature_ok(d->temperature), Q35_ERR_ARG, "temperature is 0 or at least 0.001");
        VerifyArgs a{};
        a.logits = d->logits; a.draft_logits = d->temperature == 0.0 ? nullptr : d->draft_logits;
        a.ld = d->ld; a.ldd = d->draft_ld; a.bf16 = d->dtype; a.n = n; a.k = k; a.vocab = vocab;
        a.set_temperature(d->temperature);
        a.drafts = d->drafts; a.u = d->u; a.accepted = accepted; a.tokens = tokens; a.stats = ev.verify_ws;
        OnDevice on(ev.device);
        HCK(launch_verify(a, ev.st));
    });
}

}  // extern "C"
