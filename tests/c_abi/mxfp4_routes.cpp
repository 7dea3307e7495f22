// Which kernel a product with MXFP4 weights takes, behind a plain C function for
// tests/test_routes_mxfp4.py.  Nothing here touches a GPU.
#include "mr_kernels.hpp"

// kind: 0 bf16, 1 f32, 2 MXFP4; experts 0: one matrix of `rows` tokens, else `rows`
// pairs.  out: kernel (0 few, 1 mid, 2 tiles), weight rows and rows of x of a
// workgroup, waves, stages.
extern "C" void route_mxfp4(int kind, int rows, int out_features, int in_features, int experts, int per_token, int cus, int* out) {
    mr::Mxfp4GemmParams p{};
    p.x_kind = kind;
    p.ldx = in_features;
    p.M = experts ? rows / per_token : rows;
    p.N = out_features;
    p.K = in_features;
    p.offsets = experts ? reinterpret_cast<const int32_t*>(uintptr_t(1) << 20) : nullptr;  // never dereferenced
    p.experts = experts;
    p.pairs = experts ? rows : 0;
    p.per_token = per_token;
    const mr::Mxfp4Route r = mr::mxfp4_route(p, cus);
    out[0] = r.kernel;
    out[1] = r.out;
    out[2] = r.rows;
    out[3] = r.waves;
    out[4] = r.stages;
}
