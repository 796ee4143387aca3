// What the entry points over the 4-bit cache share (q35_kv4.cpp, q35_answers.cpp): the cache's handle and the
// checks of arguments.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>
#include <vector>

#include "q35_host.h"
#include "q35_kv4.h"

struct q35_kv4 {
    q35_engine* eng = nullptr;
    int device = 0, layers = 0, lanes = 0, cap = 0, kv_heads = 0, D = 0;
    uint8_t* mem = nullptr;          // [layers][lanes][kv_heads] regions
    std::vector<int> len;            // [layers][lanes] slots held
    size_t region() const { return q35::kv4_region_bytes(D, cap); }
    size_t lane_bytes() const { return (size_t)kv_heads * region(); }
    size_t layer_bytes() const { return (size_t)lanes * lane_bytes(); }
    int& held(int layer, int lane) { return len[(size_t)layer * lanes + lane]; }
};

namespace q35 {

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

inline void check_dim(int D) { REQ(D == 64 || D == 128 || D == 256, Q35_ERR_ARG, "head_dim is 64, 128 or 256"); }

// A view of rows: 16-byte loads and stores from every (row, head).
inline HeadView view(const q35_view& v, const char* what) {
    const auto bad = [&](const char* why) { return Q35Error(Q35_ERR_ARG, std::string(what) + ": " + why); };
    if (!v.ptr) throw bad("null pointer");
    if ((uintptr_t)v.ptr % 16 || v.row_stride % 8 || v.head_stride % 8)
        throw bad("the pointer must be 16-byte aligned and the strides multiples of 8 elements");
    if (v.row_stride < 0 || v.head_stride < 0) throw bad("negative stride");
    return {v.ptr, v.row_stride, v.head_stride};
}
inline HeadView maybe_view(const q35_view& v, const char* what) { return v.ptr ? view(v, what) : HeadView{nullptr, 0, 0}; }
// An output's heads and rows must not share elements.
inline void check_out(const HeadView& v, int heads, int rows, int D, const char* what) {
    if (!v.p) return;
    const bool apart = (heads == 1 || v.head >= D) && (rows == 1 || v.row >= D) &&
                       (heads == 1 || rows == 1 || v.row >= (heads - 1) * v.head + D || v.head >= (rows - 1) * v.row + D);
    REQ(apart, Q35_ERR_ARG, std::string(what) + ": rows or heads overlap");
}

// Sequences of a call on cache c's `layer`: lanes in range (i when null); each position at most the lane's
// length for an append (which then holds pos + T slots), pos + T at most the length for a read.
inline void check_seqs(q35_kv4* c, int layer, const int32_t* lanes, const int32_t* pos, int n, int T, bool append) {
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

inline void check_cache(q35_engine* e, q35_kv4* c) {
    REQ(e && c, Q35_ERR_ARG, "null argument");
    REQ(c->eng == e, Q35_ERR_ARG, "the cache belongs to another engine");
}

inline HeadArgs head_args(const q35_heads& s, int kv_heads, int D, int n, int T, bool cached) {
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
template <class Args>
void run_heads(Args a, const int32_t* lanes, const int32_t* pos, int n, hipStream_t st) {
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
        if constexpr (std::is_same<Args, AxisHeadArgs>::value) a.axis_pos += (long long)m * a.T * a.row_step;
    }
}

}  // namespace q35
