// The host half of the 4-bit cache's entry points without a GPU: the HIP calls and launchers that
// q35_kv4.cpp makes, counted instead of run, so that its argument checks are testable on any machine.
#include <cstdlib>
#include <cstring>

#include "q35_host.h"
#include "q35_kv4.h"

struct q35_engine { int launches = 0; };
static q35_engine* g_now = nullptr;
static std::string g_text;

namespace q35 {
int guard(const std::function<void()>& f) {
    try {
        f();
        return Q35_OK;
    } catch (const Q35Error& ex) {
        g_text = ex.what();
        return ex.code;
    }
}
EngineView engine_view(q35_engine* e) {
    g_now = e;
    return {0, 64, 4096, nullptr, nullptr, nullptr};
}
static hipError_t count() {
    ++g_now->launches;
    return hipSuccess;
}
hipError_t launch_heads(HeadArgs&, int, hipStream_t) { return count(); }
hipError_t launch_attn_kv4(Kv4Attn&, int, hipStream_t) { return count(); }
hipError_t launch_kv4_copy(const Kv4Copy&, bool, hipStream_t) { return count(); }
hipError_t launch_verify(VerifyArgs&, hipStream_t) { return count(); }
}  // namespace q35

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t) { *p = std::malloc(16); return hipSuccess; }
hipError_t hipFree(void* p) { std::free(p); return hipSuccess; }
hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "stub"; }

q35_engine* stub_engine() { return new q35_engine(); }
int stub_launches(q35_engine* e) { return e->launches; }
const char* q35_last_error() { return g_text.c_str(); }
}
