// How a call of attention over a paged cache is split, behind a plain C function for
// tests/test_routes_kv.py.  Nothing here touches a GPU.
#include "mr_kernels.hpp"

// out: the form for many queries, rows of a tile, parts, keys of a part
extern "C" void route_kv(long tokens, int batch, int ragged, int kv_heads, int group, int dim, int window, long keys, int cus,
                         int* out) {
    const mr::KvAttnRoute r = mr::kv_attention_route(tokens, batch, ragged != 0, kv_heads, group, dim, window, keys, cus);
    out[0] = r.prompt;
    out[1] = r.rows;
    out[2] = r.splits;
    out[3] = r.chunk;
}
