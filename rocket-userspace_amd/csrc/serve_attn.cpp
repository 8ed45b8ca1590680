// serve_attn.cpp — which kernel a serving attention call takes.
#include "serve.h"

namespace rk {

size_t serve_attn_ws(const ServeAttn &a) { return !a.Kf && kv4_few_rows(a) ? kv4_rows_ws(a) : serve_tiles_ws(a); }

hipError_t serve_attn(const ServeAttn &a, hipStream_t s, uint64_t *blocks)
{
    return !a.Kf && kv4_few_rows(a) ? kv4_rows(a, s, blocks) : serve_tiles(a, s, blocks);
}

}  // namespace rk
