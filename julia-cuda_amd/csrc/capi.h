// What the C ABI's translation units share: errors into the caller's buffer, the scratch.
#pragma once

#include <string.h>

#include <algorithm>
#include <exception>
#include <string>

#include "../../include/julia_hip.h"
#include "kernels.h"

struct julia_hip_scratch {
    jh::Scratch s;
};

namespace jh {

inline void report(char* err, size_t len, const std::string& msg) {
    if (!err || len == 0) return;
    const size_t n = std::min(msg.size(), len - 1);
    memcpy(err, msg.data(), n);
    err[n] = 0;
}

template <typename F>
int guarded(char* err, size_t len, F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& ex) {
        report(err, len, ex.what());
    } catch (...) {
        report(err, len, "julia-hip: unknown exception");
    }
    return -1;
}

inline Scratch scratch_of(const julia_hip_scratch* s) { return s ? s->s : Scratch{}; }

}  // namespace jh
