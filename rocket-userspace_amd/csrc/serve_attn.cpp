// serve_attn.cpp — which kernel a serving attention call takes: few query rows a KV head run in
// registers, over codes (kv4_rows.hip) or fp16 keys (attn_decode.hip), more in tiles (serve_tiles.hip).
#include "attn.h"
#include "serve.h"

namespace rk {

namespace {

// The call over fp16 keys as the few-row kernel takes it.
FaLaunch rows_launch(const ServeAttn &a)
{
    FaLaunch f;
    f.Q = a.Q; f.K = a.Kf; f.Vt = a.Vf; f.O = a.out;
    f.q_hs = (long)a.n_tokens * a.dk; f.q_rs = a.dk;
    f.k_hs = a.k_hs; f.k_rs = a.dk;
    f.v_hs = (long)a.dv * a.stride; f.v_rs = a.stride;
    f.o_hs = (long)a.n_tokens * a.dv; f.o_rs = a.dv;
    f.T = a.n_tokens; f.n_kv = a.max_kv; f.dk = a.dk; f.dv = a.dv; f.n_head = a.n_head; f.gqa = a.gqa;
    f.scale = a.scale; f.softcap = a.softcap;
    f.win = true; f.window = a.window; f.sinks = a.sinks;
    f.ws = a.ws; f.ws_bytes = a.ws_bytes;
    return f;
}

}  // namespace

bool serve_few_rows(const ServeAttn &a) { return a.Kf ? flash_attn_few_rows(rows_launch(a)) : kv4_few_rows(a); }

size_t serve_attn_ws(const ServeAttn &a)
{
    if (!serve_few_rows(a)) return serve_tiles_ws(a);
    return a.Kf ? flash_attn_rows_ws(rows_launch(a)) : kv4_rows_ws(a);
}

hipError_t serve_attn(const ServeAttn &a, hipStream_t s, uint64_t *blocks)
{
    if (!serve_few_rows(a)) return serve_tiles(a, s, blocks);
    return a.Kf ? flash_attn_rows(rows_launch(a), s, blocks) : kv4_rows(a, s, blocks);
}

}  // namespace rk
