// kv8_attention.cu -- attention over 8-bit key/value caches, alone (mt_attention_kv8) and behind a
// prefix that all requests share (mt_attention_prefix_kv8).
//
// out = sum_j w_j v_j / sum_j w_j with w_j = exp(q.k_j / 8 - m), one pass with a running maximum m.
// The reference's attention_cache (Shaders.swift:500-591) reads fp32 caches of one request.
#include <cuda_fp8.h>
#include <math.h>

#include "kv8.cuh"

namespace mt {

namespace {

struct Kv8View {
    const uint8_t *k, *v;
    const float *ks, *vs;
    long long request_stride;
    int capacity, kind;
};

struct Kv8AttnArgs {
    const float* q; int ldq;
    float* out; int ldo;
    Kv8Rows rows;
    int requests, hq, hkv, window;
    Kv8View own, prefix;
    int prefix_len;
};

constexpr int AT_WARPS = 4;

__device__ __forceinline__ float2 decode2(uint32_t c, int kind) {
    if (kind == MT_KV_INT8) return make_float2((float)(int8_t)c, (float)(int8_t)(c >> 8));
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xFFFFu), __NV_E4M3)));
}

// One warp a (row, query head): 32 keys at a time, a lane a key for the scores and a lane two
// dimensions for the values.
__global__ void __launch_bounds__(AT_WARPS * 32) kv8_attention_kernel(Kv8AttnArgs a) {
    __shared__ float qs[AT_WARPS][64];
    pdl_wait();
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * AT_WARPS + warp;
    const int head = (int)(unit % a.hq);
    const long long row = unit / a.hq;
    if (row >= (long long)a.requests * a.rows.rows) return;
    const int request = (int)(row / a.rows.rows), i = (int)(row % a.rows.rows);
    const Kv8Span s = kv8_span(a.rows, request);
    if (i >= s.count) return;
    const float* q = a.q + (size_t)row * a.ldq + (size_t)head * 64;
    qs[warp][lane] = q[lane] * 0.125f;
    qs[warp][lane + 32] = q[lane + 32] * 0.125f;
    __syncwarp();
    const int p = s.pos + i;
    int first = max(a.rows.base, s.pos + s.count - a.own.capacity);
    if (a.window > 0) first = max(first, p - a.window + 1);
    const int kh = head / (a.hq / a.hkv);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int part = 0; part < 2; part++) {
        const Kv8View& c = part == 0 ? a.prefix : a.own;
        const int from = part == 0 ? 0 : first, to = part == 0 ? a.prefix_len : p + 1;
        const size_t base = (part == 0 ? 0 : (size_t)request * c.request_stride) + (size_t)kh * c.capacity;
        for (int j0 = from; j0 < to; j0 += 32) {
            const int j = j0 + lane;
            const bool on = j < to;
            const int slot = on ? (part == 0 ? j : (j - a.rows.base) % c.capacity) : 0;
            float score = -INFINITY, vs = 0.f;
            if (on) {
                const uint4* kr = reinterpret_cast<const uint4*>(c.k + (base + slot) * 64);
                float d = 0.f;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const uint4 w = kr[t];
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const float2 f = decode2(ws[u], c.kind), g = decode2(ws[u] >> 16, c.kind);
                        const float* qq = &qs[warp][t * 16 + u * 4];
                        d = fmaf(f.x, qq[0], fmaf(f.y, qq[1], fmaf(g.x, qq[2], fmaf(g.y, qq[3], d))));
                    }
                }
                score = d * c.ks[base + slot];
                vs = c.vs[base + slot];
            }
            float top = warp_max(score);
            const float mn = fmaxf(m, top);
            const float fix = mn == -INFINITY ? 1.f : expf(m - mn);
            const float w = on ? expf(score - (mn == -INFINITY ? 0.f : mn)) : 0.f;
            m = mn;
            l = l * fix + w;
            o0 *= fix;
            o1 *= fix;
            const float wv = on ? w * vs : 0.f;
            const int n = min(32, to - j0);
            for (int t = 0; t < n; t++) {
                const float x = __shfl_sync(0xffffffffu, wv, t);
                const int sl = __shfl_sync(0xffffffffu, slot, t);
                const float2 f = decode2(reinterpret_cast<const uint16_t*>(c.v + (base + sl) * 64)[lane], c.kind);
                o0 = fmaf(x, f.x, o0);
                o1 = fmaf(x, f.y, o1);
            }
        }
    }
    l = warp_sum(l);
    float* out = a.out + (size_t)row * a.ldo + (size_t)head * 64;
    out[2 * lane] = o0 / l;
    out[2 * lane + 1] = o1 / l;
}

Kv8View view(const mt_kv8_cache* c) {
    return Kv8View{c->k, c->v, c->k_scale, c->v_scale, c->request_stride, c->capacity, c->kind};
}

size_t workspace_bytes(const mt_ctx*, int prefix_len, const mt_kv8_cache* cache, int requests, int rows, int hq, int window) {
    (void)prefix_len; (void)cache; (void)requests; (void)rows; (void)hq; (void)window;
    return 0;
}

mt_status attention(mt_ctx* ctx, const char* what, void* stream, const float* q, int ldq, int requests, int rows, int hq,
                    const int32_t* positions, const int32_t* counts, int window, const mt_kv8_cache* prefix, int prefix_len,
                    const mt_kv8_cache* cache, float* out, int ldo, void* workspace, size_t have) {
    MT_REQUIRE(ctx, q && positions && out, MT_ERR_ARG, "%s: null argument", what);
    mt_status st = kv8_check_cache(ctx, what, cache, requests);
    if (st != MT_OK) return st;
    const int hkv = cache->kv_heads;
    st = kv8_check_rows(ctx, what, requests, rows, hq, hkv);
    if (st != MT_OK) return st;
    MT_REQUIRE(ctx, ldq >= hq * 64 && ldo >= hq * 64 && window >= 0, MT_ERR_SHAPE, "%s: hq %d ldq %d ldo %d window %d", what,
               hq, ldq, ldo, window);
    MT_REQUIRE(ctx, rows <= cache->capacity && (window == 0 || (long long)window + rows - 1 <= cache->capacity), MT_ERR_CAPACITY,
               "%s: %d rows, window %d, capacity %d", what, rows, window, cache->capacity);
    MT_REQUIRE(ctx, ctx, MT_ERR_ARG, "%s: null context", what);
    const size_t need = workspace_bytes(ctx, prefix_len, cache, requests, rows, hq, window);
    MT_REQUIRE(ctx, need == 0 || (workspace && have >= need && ((uintptr_t)workspace & 15u) == 0), MT_ERR_CAPACITY,
               "%s: workspace of %zu bytes (16-byte aligned), needs %zu", what, workspace ? have : (size_t)0, need);
    if (requests == 0 || rows == 0) return MT_OK;
    DeviceGuard guard(ctx->device);
    MT_REQUIRE(ctx, guard.err == cudaSuccess, MT_ERR_CUDA, "%s: %s", what, cudaGetErrorString(guard.err));
    Kv8AttnArgs a{};
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo;
    a.rows = Kv8Rows{positions, counts, rows, cache->base};
    a.requests = requests; a.hq = hq; a.hkv = hkv; a.window = window;
    a.own = view(cache);
    a.prefix = prefix_len > 0 ? view(prefix) : a.own;
    a.prefix_len = prefix_len;
    const long long blocks = ((long long)requests * rows * hq + AT_WARPS - 1) / AT_WARPS;
    MT_REQUIRE(ctx, blocks <= 0x7FFFFFFFll, MT_ERR_SHAPE, "%s: %d requests of %d rows", what, requests, rows);
    launch_k(kv8_attention_kernel, (unsigned)blocks, AT_WARPS * 32, 0, as_stream(stream), a);
    return check_launch(ctx, what);
}

}  // namespace

}  // namespace mt

using namespace mt;

extern "C" {

size_t mt_attention_kv8_workspace(const mt_ctx* ctx, const mt_kv8_cache* cache, int requests, int rows, int hq, int window) {
    return ctx && cache ? workspace_bytes(ctx, 0, cache, requests, rows, hq, window) : 0;
}

size_t mt_attention_prefix_kv8_workspace(const mt_ctx* ctx, int prefix_len, const mt_kv8_cache* cache, int requests,
                                         int rows, int hq) {
    return ctx && cache ? workspace_bytes(ctx, prefix_len, cache, requests, rows, hq, 0) : 0;
}

mt_status mt_attention_kv8(mt_ctx* ctx, void* stream, const float* q, int ldq, int requests, int rows, int hq,
                           const int32_t* positions, const int32_t* counts, int window, const mt_kv8_cache* cache,
                           float* out, int ldo, void* workspace, size_t workspace_bytes) {
    return attention(ctx, "mt_attention_kv8", stream, q, ldq, requests, rows, hq, positions, counts, window, nullptr, 0,
                     cache, out, ldo, workspace, workspace_bytes);
}

mt_status mt_attention_prefix_kv8(mt_ctx* ctx, void* stream, const float* q, int ldq, int requests, int rows, int hq,
                                  const int32_t* positions, const int32_t* counts, const mt_kv8_cache* prefix,
                                  int prefix_len, const mt_kv8_cache* cache, float* out, int ldo, void* workspace,
                                  size_t workspace_bytes) {
    const char* what = "mt_attention_prefix_kv8";
    MT_REQUIRE(ctx, prefix_len >= 0, MT_ERR_SHAPE, "%s: prefix of %d positions", what, prefix_len);
    if (prefix_len > 0) {
        mt_status st = kv8_check_cache(ctx, what, prefix, 1);
        if (st != MT_OK) return st;
        MT_REQUIRE(ctx, prefix->base == 0 && prefix_len <= prefix->capacity, MT_ERR_CAPACITY,
                   "%s: prefix of %d positions in a cache of %d from %d on", what, prefix_len, prefix->capacity, prefix->base);
    }
    MT_REQUIRE(ctx, cache && cache->base == prefix_len && (prefix_len == 0 || cache->kv_heads == prefix->kv_heads),
               MT_ERR_SHAPE, "%s: the requests' cache starts at %d behind a prefix of %d, heads %d and %d", what,
               cache ? cache->base : -1, prefix_len, cache ? cache->kv_heads : 0, prefix_len ? prefix->kv_heads : 0);
    return attention(ctx, what, stream, q, ldq, requests, rows, hq, positions, counts, 0, prefix, prefix_len, cache, out,
                     ldo, workspace, workspace_bytes);
}

}  // extern "C"
