// layer.h — launches behind rocket_fp8.h and rocket_layer.h: products of e4m3 codes with block scales (fp8_gemm.hip,
// fp8_rows.hip), their quantisation (fp8_quant.hip), block norms (add_norm.hip) and routing (moe_route.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "rocket_fp8.h"
#include "rocket_layer.h"

namespace rk {

constexpr int kF8Block = 128;        // values that share a scale
constexpr int kF8MaxK = 1 << 16;
constexpr int kNormMaxH = 1 << 14;
constexpr int kMaxExperts = 1024, kMaxTop = 32, kMaxGroups = 64;
inline int f8_blocks(int n) { return (n + kF8Block - 1) / kF8Block; }

// A group's scale and the factor to its codes, the same steps on the host and on the GPU (fp32, IEEE division).
__host__ __device__ inline float f8_amax(float a) { return a > 0x1p-100f ? a : 0x1p-100f; }
__host__ __device__ inline float f8_clamp(float v) { return v > 448.f ? 448.f : v < -448.f ? -448.f : v; }   // (NaN stays)

struct QuantF8 {
    const void *a = nullptr, *up = nullptr;   // rows, or gate and up rows (act); fp16 or fp32 (f32)
    long rs = 0;
    bool f32 = false;
    int act = 0, M = 0, K = 0;
    const int32_t *n_rows = nullptr;
    uint8_t *q = nullptr;
    float *scale = nullptr;
};
hipError_t quant_fp8(const QuantF8 &L, hipStream_t s, uint64_t *blocks);

// One product (expert_off null: n_expert 1), or experts' products.
struct GemmF8 {
    const uint8_t *A = nullptr, *B = nullptr;
    const float *sa = nullptr, *sb = nullptr;
    const int32_t *src = nullptr, *off = nullptr;
    void *C = nullptr;
    bool f16 = false;
    int M = 0, K = 0, N = 0, n_expert = 1, a_rows = 0;   // M: rows of C
    int kind = 0, slices = 1;   // the kernel, and its slices of K (gemm_fp8_plan)
    float *ws = nullptr;        // the slices' sums; without it a workgroup walks all of K
};
// Chooses the launch's kernel and slices. The bytes that `ws` has to have (0: no slices).
size_t gemm_fp8_plan(GemmF8 &L);
hipError_t gemm_fp8(const GemmF8 &L, hipStream_t s, uint64_t *blocks);

// Few rows (fp8_rows.hip): the time that they are expected to take (infinite: too many rows), and the launch.
float gemm_fp8_rows_us(const GemmF8 &L);
hipError_t gemm_fp8_rows(const GemmF8 &L, hipStream_t s, uint64_t *blocks);

struct AddNorm {
    const void *h = nullptr, *y = nullptr, *shared = nullptr;   // fp16 or fp32 (f32)
    void *h_out = nullptr;
    bool f32 = false;
    long y_rs = 0;
    const _Float16 *w_post = nullptr, *w_pre = nullptr, *gate = nullptr;
    float eps_post = -1.f, eps_pre = -1.f, alpha = 1.f;
    int gate_every = 1, M = 0, H = 0;
    int top_k = 0, rows = 0;            // experts' rows: top_k > 0, y[rows][H]
    const int32_t *slot = nullptr;
    const float *weight = nullptr;
    _Float16 *x = nullptr;
    uint8_t *xq = nullptr;
    float *x_scale = nullptr;
};
hipError_t add_norm(const AddNorm &L, hipStream_t s, uint64_t *blocks);

struct Route {
    const void *logits = nullptr;
    bool f32 = false, sigmoid = false, renorm = false;
    long rs = 0;
    const float *bias = nullptr;
    const uint8_t *active = nullptr;
    int M = 0, E = 0, n_group = 1, group_best = 1, top_group = 1, top_k = 0;
    float scale = 1.f;
    int32_t *ids = nullptr, *off = nullptr, *src = nullptr, *slot = nullptr;
    float *weight = nullptr;
    int32_t *counts = nullptr;          // route_ws() bytes of scratch
};
size_t route_ws(const Route &L);
hipError_t moe_route(const Route &L, hipStream_t s, uint64_t *blocks);

// The host paths (fd < 0): products, norms and scores in fp64, codes by the formula.
void quant_fp8_ref(const QuantF8 &L);
bool gemm_fp8_ref(const GemmF8 &L);
bool add_norm_ref(const AddNorm &L);
bool moe_route_ref(const Route &L);

}  // namespace rk
