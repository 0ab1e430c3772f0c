/*
 * What the host sides of include/eri_layers.h and include/eri_losses.h share: error messages, limits, checks of addresses
 * and strides.  Local to the file that includes it.
 */
#pragma once
#include <hip/hip_runtime.h>

#include <cstdio>

#include "../../include/eri_layers.h"

namespace {

int fail(int code, const char *msg) {
    eri_set_last_error(msg);
    return code;
}
int fail(int code, const char *call, const char *what) {
    char buf[160];
    std::snprintf(buf, sizeof buf, "%s: %s", call, what);
    return fail(code, buf);
}
int done(int hip_error, const char *call) {
    return hip_error == 0 ? 0 : fail(hip_error, call, hipGetErrorString((hipError_t)hip_error));
}

constexpr uint64_t kCountMost = 0x7fffffffull;                 // rows, columns, tokens, ids
constexpr uint64_t kStrideMost = (uint64_t)1 << 40;            // so that no offset leaves 64 bits

bool floating(int tag) { return tag == ERI_DTYPE_F32 || tag == ERI_DTYPE_BF16; }
uint32_t size_of(int tag) { return tag == ERI_DTYPE_F32 ? 4 : tag == ERI_DTYPE_BF16 ? 2 : 1; }
bool aligned(const void *p, uint32_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

/* Sets a stride of 0 to the row's length and refuses one that is shorter. */
bool stride(uint64_t *s, uint64_t cols) {
    if (*s == 0) *s = cols;
    return *s >= cols && *s <= kStrideMost;
}

#define ERI_NEED(cond, code, what) \
    do {                           \
        if (!(cond)) return fail(code, kCall, what); \
    } while (0)

} // namespace
