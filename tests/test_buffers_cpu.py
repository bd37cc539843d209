"""The env's buffers that grow together (csrc/g1_buffers.h), with a fake allocator whose n-th allocation fails: after a failure the
group owns nothing, so a later call that asks for less allocates again instead of using what was freed."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "g1.cu_b200", "csrc")

HARNESS = r"""
#include <stdio.h>
#include <stdlib.h>
#include <set>
typedef int cudaError_t;
enum { cudaSuccess = 0, cudaErrorMemoryAllocation = 2 };
static std::set<void*> live;
static int fail_at = -1, last = 0, bad_free = 0, frees = 0;
static cudaError_t cudaMalloc(void** p, size_t n) {
    if (fail_at >= 0 && fail_at-- == 0) { last = cudaErrorMemoryAllocation; return last; }
    *p = malloc(n ? n : 1);
    live.insert(*p);
    return cudaSuccess;
}
static cudaError_t cudaFree(void* p) {
    if (!p) return cudaSuccess;
    ++frees;
    if (!live.erase(p)) ++bad_free;
    else free(p);
    return cudaSuccess;
}
static cudaError_t cudaGetLastError() { int e = last; last = 0; return e; }
#include "g1_buffers.h"

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    for (int at = 0; at < 3; ++at) {
        float *a = nullptr, *b = nullptr;
        short* c = nullptr;
        size_t n = 0, w = 0;
        auto ask = [&](size_t N, size_t W) {
            return grow({{&n, N}, {&w, W}}, {grow_buf(&a, N), grow_buf(&b, N * W), grow_buf(&c, W)});
        };
        CHECK(ask(10, 8) == cudaSuccess && n == 10 && w == 8 && live.size() == 3);
        float* was = a;
        CHECK(ask(10, 4) == cudaSuccess && a == was && n == 10 && w == 8);   // large enough: nothing moves
        fail_at = at;
        CHECK(ask(10, 100) == cudaErrorMemoryAllocation);
        CHECK(!a && !b && !c && n == 0 && w == 0 && live.empty() && last == 0);
        fail_at = -1;
        CHECK(ask(10, 8) == cudaSuccess && a && b && c && live.size() == 3 && n == 10 && w == 8);  // what fitted before
        CHECK(ask(4, 9) == cudaSuccess && n == 4 && w == 9);
        CHECK(ask(10, 8) == cudaSuccess && n == 10 && w == 8);
        cudaFree(a); cudaFree(b); cudaFree(c);
        CHECK(live.empty() && bad_free == 0);
    }
    printf("BUFFERS OK\n");
    return 0;
}
"""


def test_a_failed_allocation_leaves_no_stale_buffers(tmp_path):
    src, exe = tmp_path / "buffers.cpp", tmp_path / "buffers"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=address", "-I", CSRC, str(src), "-o", str(exe)], check=True,
                   capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "BUFFERS OK" in r.stdout, r.stdout + r.stderr


def test_every_buffer_that_grows_goes_through_it():
    """No buffer of an env is freed and allocated anew by hand."""
    with open(os.path.join(CSRC, "g1_env.cu")) as f:
        body = f.read()
    lo, hi = body.index("void g1_env_destroy(void* h)"), body.index("void* g1_env_create_ex(")
    outside = body[:hi] + body[lo + body[lo:].index("\n}\n"):]
    for name in ("Xb", "Hb[0]", "Hb[1]", "HD", "Wb", "Bf", "LS", "Wvb", "Bvf", "HDv", "tf_img", "WT"):
        assert f"cudaFree(E->{name})" not in outside and f"cudaMalloc(&E->{name}," not in outside, name
