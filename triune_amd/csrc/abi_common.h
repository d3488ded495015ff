// abi_common.h -- argument checks that the C entries of abi_ssm.hip and abi_decay.hip share.  Internal to libtriune_hip.
#pragma once

#include "../../include/triune_hip.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <initializer_list>

namespace {

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxGrid = 0x7fffffff;

size_t align_up(size_t x) { return (x + 255) / 256 * 256; }
int status(hipError_t e) { return e == hipSuccess ? TRIUNE_OK : TRIUNE_ERR_LAUNCH; }
bool dtype_ok(int dt) { return dt == TRIUNE_DT_F32 || dt == TRIUNE_DT_BF16 || dt == TRIUNE_DT_F16; }
bool aligned(const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) % (dt == TRIUNE_DT_F32 ? 4 : 2) == 0; }

// Compute units of the current device, asked once per device (MI355X: 256).
int compute_units() {
    static std::atomic<int> cache[kMaxDevices];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
        (void)hipGetLastError();
        return 256;
    }
    int n = cache[dev].load(std::memory_order_relaxed);
    if (n > 0) return n;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Sequences and tokens within the numbers that the plans multiply.
bool tokens_ok(int64_t n, int64_t T) { return n >= 0 && n <= kMaxGrid && T >= 0 && T < (1 << 30); }

// Whether n times `blocks` workgroups are a grid: 31 bits of workgroups and 32 of threads.
bool grid_ok(int64_t n, int64_t blocks, int threads) {
    const int64_t by_threads = (int64_t)0xffffffff / threads, most = by_threads < kMaxGrid ? by_threads : kMaxGrid;
    return n <= most / blocks;
}

int check_ws(const void* ws, size_t have, size_t need) {
    if (need == 0) return TRIUNE_OK;
    if (!ws || have < need) return TRIUNE_ERR_WORKSPACE;
    return reinterpret_cast<uintptr_t>(ws) % 16 ? TRIUNE_ERR_LAYOUT : TRIUNE_OK;
}

bool all_aligned(int dt, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (!aligned(p, dt)) return false;
    return true;
}

}  // namespace
