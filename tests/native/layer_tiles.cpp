// layer_tiles.cpp — on the fake runtime of fake_hip.h: which kernels the products of rocket_fp8.h launch. A line of standard input is a
// call, "fp16 grouped gathered experts rows K N" (the first three 0 or 1); its line of output, the kernels' names. Built and run by
// tests/layertiles.py.
#include "fake_hip.h"

#include <cxxabi.h>
#include <stdio.h>

#include "rocket_fp8.h"
#include "rocket_hip.h"
#include "rocket_npu.h"

static char *const at = reinterpret_cast<char *>((uintptr_t)1 << 44);   // operands, 2^40 apart, that no kernel reads here
template <class T> static T *p(size_t i) { return reinterpret_cast<T *>(at + (i << 40)); }

int main()
{
    const int fd = rocket_open();
    if (fd < 0 || rocket_hip_set_mode(fd, ROCKET_HIP_ASYNC | ROCKET_HIP_DEVICE_OPERANDS)) return 1;
    auto &f = fake::st();
    int f16, grouped, gathered, E, rows, K, N;
    while (scanf("%d %d %d %d %d %d %d", &f16, &grouped, &gathered, &E, &rows, &K, &N) == 7) {
        f.launches.clear();
        const uint8_t *const A = p<uint8_t>(0), *const B = p<uint8_t>(1);
        const float *const sa = p<float>(2), *const sb = p<float>(3);
        const int32_t *const src = gathered ? p<int32_t>(4) : nullptr, *const off = p<int32_t>(5);
        int rc;
        if (grouped)
            rc = f16 ? rocket_matmul_fp8_block_grouped_f16out(fd, E, rows, rows, K, N, A, sa, src, off, B, sb, p<_Float16>(6))
                     : rocket_matmul_fp8_block_grouped(fd, E, rows, rows, K, N, A, sa, src, off, B, sb, p<float>(6));
        else
            rc = f16 ? rocket_matmul_fp8_block_f16out(fd, rows, K, N, A, sa, B, sb, p<_Float16>(6)) : rocket_matmul_fp8_block(fd, rows, K, N, A, sa, B, sb, p<float>(6));
        if (rc) {
            fprintf(stderr, "layer_tiles: a call returned %d\n", rc);
            return 1;
        }
        for (const auto &l : f.launches) {
            char *const name = abi::__cxa_demangle(l.c_str(), nullptr, nullptr, nullptr);
            printf("%s;", name ? name : l.c_str());
            free(name);
        }
        printf("%d\n", (int)f.block.x);
    }
    rocket_close(fd);
    return 0;
}
