// serve_check.cpp — on the fake runtime of fake_hip.h: which operands of rocket_serve.h's calls are used in place (a call
// that stages one takes scratch of the handle and waits for its stream, which a captured call may not), and which calls
// over the cache split their keys. Built and run by
// tests/test_serve_staging.py. Exit status 0 when every check passes.
#include "fake_hip.h"

#include <stdio.h>

#include "rocket_hip.h"
#include "rocket_npu.h"
#include "rocket_serve.h"

static int g_fail = 0;
#define CHECK(c)                                                                                       \
    do {                                                                                               \
        if (!(c)) {                                                                                    \
            fprintf(stderr, "serve_check: %s:%d: CHECK(%s) failed\n", __FILE__, __LINE__, #c);         \
            g_fail++;                                                                                  \
        }                                                                                              \
    } while (0)

// Operands: addresses that no kernel reads here.
static char *const at = reinterpret_cast<char *>((uintptr_t)1 << 40);
template <class T> static T *p(size_t off) { return reinterpret_cast<T *>(at + off); }

// A first call of a handle, captured: it launches, and neither allocates nor waits.
template <class F> static void in_place(const char *what, F call)
{
    auto &f = fake::st();
    const int fd = rocket_open();
    CHECK(fd >= 0);
    CHECK(rocket_hip_set_mode(fd, ROCKET_HIP_ASYNC | ROCKET_HIP_DEVICE_OPERANDS) == 0);
    f.launches.clear();
    const size_t live = f.live.size();
    const int syncs = f.syncs;
    f.capturing = true;
    const int rc = call(fd);
    f.capturing = false;
    if (rc || f.launches.size() != 1 || f.live.size() != live || f.syncs != syncs) {
        fprintf(stderr, "serve_check: %s: status %d, %zu launches, %zu allocations, %d waits\n", what, rc, f.launches.size(), f.live.size() - live, f.syncs - syncs);
        g_fail++;
    }
    rocket_close(fd);
}

// Launches of an eager attention call over the cache: 1, or 2 where its keys are split and merged.
static size_t launches(int seqs, int heads, int dim, int rows, int max_kv)
{
    auto &f = fake::st();
    const int fd = rocket_open();
    CHECK(rocket_hip_set_mode(fd, ROCKET_HIP_ASYNC | ROCKET_HIP_DEVICE_OPERANDS) == 0);
    const rocket_kv4_shape sh = {seqs, heads, dim, dim, max_kv};
    f.launches.clear();
    CHECK(rocket_kv4_attn_fp16(fd, &sh, at + ((size_t)1 << 36), 0, seqs, rows, max_kv, heads, 0.1f, 0.f, 0, 0, p<_Float16>(0), p<int32_t>((size_t)1 << 35),
                               p<_Float16>((size_t)1 << 34)) == 0);
    const size_t n = f.launches.size();
    rocket_close(fd);
    return n;
}

int main()
{
    typedef _Float16 H;
    // keys are split where that saves more than the merge costs: not many rows of short sequences
    CHECK(launches(32, 8, 64, 64, 300) == 1 && launches(16, 8, 128, 24, 300) == 1 && launches(32, 8, 64, 64, 1000) == 1 && launches(1, 8, 64, 1, 300) == 1);
    CHECK(launches(1, 8, 256, 1, 3000) == 2 && launches(1, 8, 128, 64, 2000) == 2 && launches(16, 8, 64, 24, 4000) == 2 && launches(32, 2, 64, 64, 3000) == 2);
    const rocket_kv4_shape sh = {8, 2, 64, 64, 400};
    H *const X = p<H>(0), *const Y = p<H>(1 << 20), *const Z = p<H>(2 << 20);
    char *const cache = at + (16 << 20);
    // lengths of places 1 and 2 of a batch's array, positions of its rows 1 and 2: the kernels read them one by one
    for (size_t i = 0; i < 4; i++) {
        int32_t *const ints = p<int32_t>((8 << 20) + 4 * i);
        in_place("append", [&](int fd) { return rocket_kv4_append_fp16(fd, &sh, cache, 1, 2, 1, X, 128, 64, 64, X, 128, 64, 64, ints); });
        in_place("read", [&](int fd) { return rocket_kv4_read_fp16(fd, &sh, cache, 1, 2, 1, ints, Y, Z); });
        for (int T : {1, 20, 90})
            in_place("attention", [&](int fd) { return rocket_kv4_attn_fp16(fd, &sh, cache, 1, 2, T, 400, 4, 0.1f, 0.f, 0, 0, X, ints, Y); });
        in_place("rotation", [&](int fd) {
            return rocket_qk_norm_rope_fp16(fd, 2, 1, 4, 2, 64, 64, 0, 1e-6f, X, 384, X + 256, 384, nullptr, nullptr, p<float>(4 << 20), ints, Y, Z);
        });
    }
    if (g_fail) return 1;
    printf("all checks passed\n");
    return 0;
}
