// Errors and the engine's handles, shared by the host sources of the C ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <functional>
#include <stdexcept>
#include <string>

#include "../../include/q35.h"

namespace q35 {

struct Q35Error : std::runtime_error {
    int code;
    Q35Error(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

// Runs f and turns what it throws into a status and the calling thread's error text.
int guard(const std::function<void()>& f);

// What the entry points outside q35_engine.cpp use of an engine.
struct EngineView {
    int device, max_rows, max_ctx;
    hipStream_t st;
    float* kv4_part;
    double* verify_ws;
};
EngineView engine_view(q35_engine* e);

}  // namespace q35

#define HCK(x)                                                                              \
    do {                                                                                    \
        hipError_t _e = (x);                                                                \
        if (_e != hipSuccess)                                                               \
            throw q35::Q35Error(Q35_ERR_HIP, std::string(#x) + ": " + hipGetErrorString(_e)); \
    } while (0)
#define REQ(cond, code, msg)                                  \
    do {                                                      \
        if (!(cond)) throw q35::Q35Error((code), (msg));      \
    } while (0)
