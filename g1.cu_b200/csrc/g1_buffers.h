// g1_buffers.h -- device buffers that an env keeps between calls and that grow together with what is asked of it.
//
// A group is its buffers and the capacities that say what they were allocated for.  While it is being allocated anew the
// capacities are 0, and they are set only once every allocation has succeeded: after a failed one the group owns nothing,
// and the next call allocates again instead of taking freed memory for buffers that are large enough.
#pragma once
#include <stddef.h>
#include <initializer_list>

struct GrowCap {
    size_t* have;
    size_t need;
};
struct GrowBuf {
    void** p;
    size_t bytes;
};
template <class T>
static inline GrowBuf grow_buf(T** p, size_t n) { return {reinterpret_cast<void**>(p), n * sizeof(T)}; }

static inline cudaError_t grow(std::initializer_list<GrowCap> caps, std::initializer_list<GrowBuf> bufs) {
    bool enough = true;
    for (const GrowCap& c : caps) enough = enough && *c.have >= c.need;
    if (enough) return cudaSuccess;
    for (const GrowCap& c : caps) *c.have = 0;
    auto release = [&]() {
        for (const GrowBuf& b : bufs) {
            cudaFree(*b.p);
            *b.p = nullptr;
        }
    };
    release();
    for (const GrowBuf& b : bufs) {
        const cudaError_t e = cudaMalloc(b.p, b.bytes);
        if (e != cudaSuccess) {
            *b.p = nullptr;
            release();
            (void)cudaGetLastError();  // returned here; the next launch's check is not to find it
            return e;
        }
    }
    for (const GrowCap& c : caps) *c.have = c.need;
    return cudaSuccess;
}
