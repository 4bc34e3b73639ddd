// paged_check.cuh -- the argument checks that the paged cache's C entry points share.
#pragma once

#include <atomic>
#include <initializer_list>

#include "common.cuh"

#define BML_API extern "C" __attribute__((visibility("default")))

namespace bml {
bml_status api_fail(bml_status code, const char *fmt, ...);
bml_status api_ok();
bml_status api_cuda_fail(cudaError_t e, const char *where);
}  // namespace bml

namespace {

using bml::api_fail;

int sm_count(int device) {
    static std::atomic<int> known[64];
    const bool keep = device >= 0 && device < 64;
    if (keep && known[device].load(std::memory_order_relaxed) > 0) return known[device].load(std::memory_order_relaxed);
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        return 148;
    }
    if (keep) known[device].store(n, std::memory_order_relaxed);
    return n;
}

int this_device() {
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess) {
        (void)cudaGetLastError();
        d = 0;
    }
    return d;
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool valid_dtype(int t) { return t == BML_F32 || t == BML_F16 || t == BML_BF16; }

// log2 of a page size, or -1
int page_shift(uint32_t page_size) {
    for (int s = 4; s <= 10; ++s)
        if (page_size == 1u << s) return s;
    return -1;
}

bml_status check_pages(uint32_t page_size, uint32_t max_pages, const char *fn) {
    if (page_shift(page_size) < 0) return api_fail(BML_E_INVALID, "%s: page_size %u is not a power of two from 16 to 1024", fn, page_size);
    if (max_pages == 0 || (uint64_t)max_pages * page_size >= (1ull << 31))
        return api_fail(BML_E_INVALID, "%s: %u pages of %u positions a request", fn, max_pages, page_size);
    return BML_OK;
}

bml_status ints(const char *fn, std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (!p || !aligned(p, 4)) return api_fail(BML_E_INVALID, "%s: null or misaligned int32 array", fn);
    return BML_OK;
}

// Whether an array that a call writes overlaps one that it reads: its CTAs do
// not wait for one another.
struct Span {
    const void *p;
    uint64_t bytes;
};
bool overlap(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    for (const Span &w : written)
        for (const Span &r : read) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(w.p), b = reinterpret_cast<uintptr_t>(r.p);
            if (a && b && a < b + r.bytes && b < a + w.bytes) return true;
        }
    return false;
}
// Whether two of the arrays that a call writes overlap.
bool overlap(std::initializer_list<Span> written) {
    for (const Span *a = written.begin(); a != written.end(); ++a)
        for (const Span *b = a + 1; b != written.end(); ++b)
            if (overlap({*a}, {*b})) return true;
    return false;
}

}  // namespace
