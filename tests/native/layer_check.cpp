// layer_check.cpp — on the fake runtime of fake_hip.h: what the calls of rocket_fp8.h and rocket_layer.h launch, which operands they use in
// place, what a captured call may take of the handle's scratch, and that results are staged in and out whole. Built and
// run by tests/test_layer_staging.py. Exit status 0 when every check passes.
#include "fake_hip.h"

#include <stdio.h>

#include "rocket_fp8.h"
#include "rocket_hip.h"
#include "rocket_layer.h"
#include "rocket_npu.h"

static int g_fail = 0;
#define CHECK(c)                                                                                       \
    do {                                                                                               \
        if (!(c)) {                                                                                    \
            fprintf(stderr, "layer_check: %s:%d: CHECK(%s) failed\n", __FILE__, __LINE__, #c);         \
            g_fail++;                                                                                  \
        }                                                                                              \
    } while (0)

typedef _Float16 H;

// Operands: addresses that no kernel reads here.
static char *const at = reinterpret_cast<char *>((uintptr_t)1 << 40);
template <class T> static T *p(size_t mib, size_t off = 0) { return reinterpret_cast<T *>(at + (mib << 20) + off); }

static int device_handle()
{
    const int fd = rocket_open();
    CHECK(fd >= 0);
    CHECK(rocket_hip_set_mode(fd, ROCKET_HIP_ASYNC | ROCKET_HIP_DEVICE_OPERANDS) == 0);
    return fd;
}

// A call of the handle, captured or not: `launches` kernels, and captured neither allocation nor wait.
template <class F> static void runs(const char *what, int fd, bool captured, size_t launches, F call)
{
    auto &f = fake::st();
    f.launches.clear();
    const size_t live = f.live.size();
    const int syncs = f.syncs;
    f.capturing = captured;
    const int rc = call(fd);
    f.capturing = false;
    if (rc || f.launches.size() != launches || (captured && (f.live.size() != live || f.syncs != syncs))) {
        fprintf(stderr, "layer_check: %s: status %d, %zu launches, %zu allocations, %d waits\n", what, rc, f.launches.size(), f.live.size() - live, f.syncs - syncs);
        g_fail++;
    }
}
template <class F> static void first(const char *what, F call)   // captured, of a fresh handle: one launch
{
    const int fd = device_handle();
    runs(what, fd, true, 1, call);
    rocket_close(fd);
}

int main()
{
    auto &f = fake::st();
    uint8_t *const A = p<uint8_t>(0), *const B = p<uint8_t>(1024);
    float *const sa = p<float>(2048), *const sb = p<float>(2112);
    H *const C = p<H>(3072);

    // a long K of few rows: one launch where there is no scratch, the slices and their join where there is
    const auto sliced = [&](int fd) { return rocket_matmul_fp8_block_f16out(fd, 200, 4096, 256, A, sa, B, sb, C); };
    first("product", sliced);
    int fd = device_handle();
    runs("product, eager", fd, false, 2, sliced);
    runs("product, captured after it", fd, true, 2, sliced);
    rocket_close(fd);
    for (int M : {1, 16, 17, 300, 5000}) first("product", [&](int h) { return rocket_matmul_fp8_block(h, M, 1024, 4096, A, sa, B, sb, p<float>(3072)); });

    for (size_t off = 0; off < 16; off += 4) {
        int32_t *const ints = p<int32_t>(4096, off), *const more = p<int32_t>(4100, off);
        float *const w = p<float>(4104, off);
        for (int rows : {8, 96, 4000})
            first("experts", [&](int h) { return rocket_matmul_fp8_block_grouped_f16out(h, 16, rows, 500, 512, 384, A, sa, ints, more, B, sb, C); });
        first("gated rows", [&](int h) { return rocket_quantize_glu_fp8_fp16(h, 100, 256, p<H>(0), p<H>(0) + 256, 512, 3, ints, B, sa); });
        first("experts' sum", [&](int h) {
            return rocket_moe_add_norm_fp16(h, 9, 512, p<H>(0), 40, 4, p<H>(64), ints, w, nullptr, nullptr, -1.f, nullptr, 1, 1.f, nullptr, 1e-6f, p<H>(0), C, B, sa);
        });
        const auto route = [&](int M, bool plan) {
            return [=](int h) {
                return rocket_moe_route_f32(h, M, 64, p<float>(0, off), 65, ROCKET_ROUTE_SOFTMAX, nullptr, 1, 1, 1, 6, 1, 1.f, p<uint8_t>(8, 1), ints, w, plan ? more : nullptr,
                                            plan ? more + 256 : nullptr, plan ? more + 65536 : nullptr);
            };
        };
        first("routing", route(32, true));
        first("routing without a plan", route(5000, false));
        // more tokens with a plan need scratch, which a fresh handle's captured call cannot have
        const int r = device_handle();
        f.launches.clear();
        f.capturing = true;
        CHECK(route(33, true)(r) != 0 && f.launches.empty());
        f.capturing = false;
        runs("routing, eager", r, false, 3, route(33, true));
        runs("routing, captured after it", r, true, 3, route(33, true));
        rocket_close(r);
    }

    // results that a call may leave in part: staged in and out whole, from host memory and from misaligned device memory
    fd = rocket_open();
    void *mem = nullptr;
    CHECK(hipMalloc(&mem, 1 << 16) == hipSuccess);
    static uint8_t a[16 * 128], b[2 * 8 * 128];
    static float s[64];
    static float host[16 * 8];
    const int32_t off[3] = {0, 3, 5};
    for (float *c : {host, reinterpret_cast<float *>(static_cast<char *>(mem) + 4)}) {
        for (int i = 0; i < 16 * 8; i++) c[i] = (float)i;
        CHECK(rocket_matmul_fp8_block_grouped(fd, 2, 16, 16, 128, 8, a, s, nullptr, off, b, s, c) == 0);
        for (int i = 0; i < 16 * 8; i++) CHECK(c[i] == (float)i);
    }
    CHECK(hipFree(mem) == hipSuccess);
    rocket_close(fd);
    if (g_fail) return 1;
    printf("all checks passed\n");
    return 0;
}
