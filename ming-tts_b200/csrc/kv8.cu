// kv8.cu -- writing and reading the 8-bit key/value cache (mt_rope_cache_kv8, mt_kv8_read).
//
// A cache row is the 64 values of one head at one position: one-byte codes and one fp32 scale. The
// reference has fp32 caches only (Qwen.swift:7-26, rope_cache Shaders.swift:456-486).
#include <cuda_fp8.h>
#include <math.h>

#include "kv8.cuh"

namespace mt {

mt_status kv8_check_cache(mt_ctx* ctx, const char* what, const mt_kv8_cache* c, int requests) {
    MT_REQUIRE(ctx, c && c->k && c->v && c->k_scale && c->v_scale, MT_ERR_ARG, "%s: null cache", what);
    MT_REQUIRE(ctx, c->kind == MT_KV_INT8 || c->kind == MT_KV_E4M3, MT_ERR_ARG, "%s: cache kind %d", what, c->kind);
    MT_REQUIRE(ctx, c->kv_heads > 0 && c->capacity > 0 && c->capacity <= (1 << 30) && c->base >= 0 &&
                        (long long)c->kv_heads * c->capacity <= c->request_stride,
               MT_ERR_SHAPE, "%s: cache of %d heads x %d positions from %d on, request stride %lld", what, c->kv_heads,
               c->capacity, c->base, c->request_stride);
    MT_REQUIRE(ctx, requests <= 1 || c->request_stride <= (1ll << 55) / requests, MT_ERR_SHAPE, "%s: request stride %lld",
               what, c->request_stride);
    MT_REQUIRE(ctx, (((uintptr_t)c->k | (uintptr_t)c->v) & 15u) == 0 &&
                        (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3u) == 0,
               MT_ERR_ARG, "%s: codes need 16-byte alignment, scales 4-byte", what);
    return MT_OK;
}

mt_status kv8_check_rows(mt_ctx* ctx, const char* what, int requests, int rows, int hq, int hkv) {
    MT_REQUIRE(ctx, requests >= 0 && rows >= 0 && (long long)requests * rows <= 0x7FFFFFFFll, MT_ERR_SHAPE,
               "%s: %d requests of %d rows", what, requests, rows);
    MT_REQUIRE(ctx, hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 1024, MT_ERR_SHAPE, "%s: hq %d hkv %d", what, hq, hkv);
    return MT_OK;
}

namespace {

constexpr int AP_THREADS = 256;
constexpr int AP_MAX_ROWS = 8;  // rows of a block: their 32 angles each are one per thread

struct AppendArgs {
    const float* qkv; int ldq;
    float* q_out; int ldqo;
    Kv8Rows rows;
    int total;           // requests * rows
    int hq, hkv;
    int block_rows;      // rows per block, <= AP_MAX_ROWS
    bool vec;            // 16-byte loads and stores of the fp32 rows
    const float* inv_freq;
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    long long request_stride;
    int capacity;
};

__device__ __forceinline__ float4 load4(const float* p, bool vec) {
    if (vec) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ void store4(float* p, float4 x, bool vec) {
    if (vec) {
        *reinterpret_cast<float4*>(p) = x;
    } else {
        p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w;
    }
}

// x / scale as a float that rounds to a coarser grid as the exact quotient does: the rounded quotient,
// moved by one unit to the neighbour with an odd last bit where the division left a remainder. No
// coarser value and no border between two such values is odd, so a second rounding cannot be caught
// on a tie that the first one made.
__device__ __forceinline__ float quotient_odd(float x, float scale) {
    const float q = __fdiv_rn(x, scale);
    const float rest = fmaf(-q, scale, x);  // exact: its sign is the remainder's
    const uint32_t u = __float_as_uint(q);
    if (rest == 0.f || (u & 1u)) return q;
    return __uint_as_float((rest > 0.f) == (x > 0.f) ? u + 1u : u - 1u);
}

template <int KIND>
__device__ __forceinline__ uint32_t encode4(float4 x, float scale) {
    const float a = quotient_odd(x.x, scale), b = quotient_odd(x.y, scale), c = quotient_odd(x.z, scale),
                d = quotient_odd(x.w, scale);
    if (KIND == MT_KV_INT8) {
        auto code = [](float q) { return (uint32_t)(uint8_t)(int8_t)min(127, max(-127, __float2int_rn(q))); };
        return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// RoPE, quantisation and the cache write. A block takes block_rows rows: first their angles, one
// thread each, in 64 bits (a position of 10^5 leaves an fp32 angle with 2 digits less, and a code is
// the same for every caller only if the rotated key is: rounding it once from 64 bits makes it so),
// then every head: 8 lanes a head, lane j the pairs (4j .. 4j+3, +32), so that loads and stores of
// a head are whole 128-byte lines and a code row is 16 words.
template <int KIND>
__global__ void __launch_bounds__(AP_THREADS) rope_cache_kv8_kernel(AppendArgs a) {
    __shared__ double turn[AP_MAX_ROWS][2][32];  // cos, sin
    __shared__ int place[AP_MAX_ROWS];           // slot, or -1: padding
    __shared__ int owner[AP_MAX_ROWS];           // request
    pdl_wait();
    pdl_launch();
    const int row0 = blockIdx.x * a.block_rows;
    const int n = min(a.block_rows, a.total - row0);
    if (threadIdx.x < n * 32) {
        const int i = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int request = (row0 + i) / a.rows.rows, at = (row0 + i) - request * a.rows.rows;
        const Kv8Span s = kv8_span(a.rows, request);
        const bool live = at < s.count;
        if (lane == 0) {
            place[i] = live ? (s.pos + at - a.rows.base) % a.capacity : -1;
            owner[i] = request;
        }
        if (live) {
            double sn, cs;
            sincos((double)(s.pos + at) * (double)a.inv_freq[lane], &sn, &cs);
            turn[i][0][lane] = cs;
            turn[i][1][lane] = sn;
        }
    }
    __syncthreads();
    const int vecs = a.hq + 2 * a.hkv;
    const int j = threadIdx.x & 7;
    // Whole warps run every iteration (the scale is a maximum over 8 lanes).
    for (int u = threadIdx.x >> 3; u < ((n * vecs + 3) & ~3); u += AP_THREADS / 8) {
        const int i = min(u / vecs, n - 1), head = u - (u / vecs) * vecs;
        const int slot = place[i];
        const bool on = u < n * vecs && slot >= 0;
        const float* src = a.qkv + (size_t)(row0 + i) * a.ldq + (size_t)head * 64 + 4 * j;
        float4 x0 = make_float4(0.f, 0.f, 0.f, 0.f), x1 = x0;
        if (on) {
            x0 = load4(src, a.vec);
            x1 = load4(src + 32, a.vec);
        }
        if (on && head < a.hq + a.hkv) {
            const double2* cs = reinterpret_cast<const double2*>(&turn[i][0][4 * j]);
            const double2* sn = reinterpret_cast<const double2*>(&turn[i][1][4 * j]);
            const double2 c0 = cs[0], c1 = cs[1], s0 = sn[0], s1 = sn[1];
            if (head < a.hq) {  // queries: 32-bit products of the exact angle's cosine and sine
                auto rot = [](float& p, float& q, double c, double s) {
                    const float cf = (float)c, sf = (float)s, r = p * cf - q * sf;
                    q = q * cf + p * sf;
                    p = r;
                };
                rot(x0.x, x1.x, c0.x, s0.x); rot(x0.y, x1.y, c0.y, s0.y);
                rot(x0.z, x1.z, c1.x, s1.x); rot(x0.w, x1.w, c1.y, s1.y);
                float* dst = a.q_out + (size_t)(row0 + i) * a.ldqo + (size_t)head * 64 + 4 * j;
                store4(dst, x0, a.vec);
                store4(dst + 32, x1, a.vec);
            } else {
                auto rot = [](float& p, float& q, double c, double s) {
                    const double pd = p, qd = q;
                    p = (float)(pd * c - qd * s);
                    q = (float)(qd * c + pd * s);
                };
                rot(x0.x, x1.x, c0.x, s0.x); rot(x0.y, x1.y, c0.y, s0.y);
                rot(x0.z, x1.z, c1.x, s1.x); rot(x0.w, x1.w, c1.y, s1.y);
            }
        }
        // max|x| over the head's 8 lanes as bit patterns: those of NaN and infinity are the largest.
        const float m0 = fmaxf(fmaxf(fabsf(x0.x), fabsf(x0.y)), fmaxf(fabsf(x0.z), fabsf(x0.w)));
        const float m1 = fmaxf(fmaxf(fabsf(x1.x), fabsf(x1.y)), fmaxf(fabsf(x1.z), fabsf(x1.w)));
        const float sum = fabsf(x0.x) + fabsf(x0.y) + fabsf(x0.z) + fabsf(x0.w) + fabsf(x1.x) + fabsf(x1.y) +
                          fabsf(x1.z) + fabsf(x1.w);  // NaN if any is (fmaxf drops NaN)
        uint32_t top = sum != sum ? 0x7FFFFFFFu : __float_as_uint(fmaxf(m0, m1));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (!on || head < a.hq) continue;
        const bool value = head >= a.hq + a.hkv;
        const int kh = head - a.hq - (value ? a.hkv : 0);
        const size_t at = (size_t)owner[i] * a.request_stride + (size_t)kh * a.capacity + slot;
        float scale = __fdiv_rn(__uint_as_float(top), KIND == MT_KV_INT8 ? 127.f : 448.f);
        uint32_t w0 = 0, w1 = 0;
        if (top >= 0x7F800000u) {
            scale = __uint_as_float(0x7FC00000u);
        } else if (scale < 1.17549435e-38f) {
            scale = 0.f;
        } else {
            w0 = encode4<KIND>(x0, scale);
            w1 = encode4<KIND>(x1, scale);
        }
        uint32_t* codes = reinterpret_cast<uint32_t*>((value ? a.v : a.k) + at * 64);
        codes[j] = w0;
        codes[8 + j] = w1;
        if (j == 0) (value ? a.v_scale : a.k_scale)[at] = scale;
    }
}

constexpr int RD_THREADS = 256;
constexpr int RD_ROWS = 64;  // rows of one (request, head) per block

struct ReadArgs {
    Kv8Rows rows;
    int hkv, capacity, tiles, out_capacity;
    long long request_stride;
    const uint8_t* codes[2];
    const float* scale[2];
    float* out[2];
};

// Sixteen lanes a row: four codes in, one 16-byte store out, so that a warp's stores are two whole rows.
// Bounded by the fp32 stores; the eight loads of a thread (four rows of keys, four of values) are
// issued before the first is used.
template <int KIND>
__global__ void __launch_bounds__(RD_THREADS) kv8_read_kernel(ReadArgs a) {
    pdl_wait();
    pdl_launch();
    const int tile = blockIdx.x % a.tiles, unit = blockIdx.x / a.tiles;
    const int head = unit % a.hkv, request = unit / a.hkv;
    const Kv8Span s = kv8_span(a.rows, request);
    const int lane = threadIdx.x & 15;
    const size_t from = (size_t)request * a.request_stride + (size_t)head * a.capacity;
    uint32_t w[2][RD_ROWS / 16];
    float sc[2][RD_ROWS / 16];
#pragma unroll
    for (int i = 0; i < RD_ROWS / 16; i++) {
        const int row = tile * RD_ROWS + i * 16 + (threadIdx.x >> 4);
        const size_t at = from + (row < s.count ? (s.pos + row - a.rows.base) % a.capacity : 0);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const bool on = row < s.count && a.out[t];
            w[t][i] = on ? reinterpret_cast<const uint32_t*>(a.codes[t] + at * 64)[lane] : 0u;
            sc[t][i] = on ? a.scale[t][at] : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < RD_ROWS / 16; i++) {
        const int row = tile * RD_ROWS + i * 16 + (threadIdx.x >> 4);
        if (row >= s.count) break;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            if (!a.out[t]) continue;
            float4 x;
            const uint32_t c = w[t][i];
            if (KIND == MT_KV_INT8) {
                x = make_float4((float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)(int8_t)(c >> 24));
            } else {
                const __half2 lo = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xFFFFu), __NV_E4M3));
                const __half2 hi = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3));
                const float2 f = __half22float2(lo), g = __half22float2(hi);
                x = make_float4(f.x, f.y, g.x, g.y);
            }
            x.x *= sc[t][i]; x.y *= sc[t][i]; x.z *= sc[t][i]; x.w *= sc[t][i];
            reinterpret_cast<float4*>(a.out[t] + ((size_t)unit * a.out_capacity + row) * 64)[lane] = x;
        }
    }
}

}  // namespace

}  // namespace mt

using namespace mt;

extern "C" mt_status mt_rope_cache_kv8(mt_ctx* ctx, void* stream, const float* qkv, int ldq, int requests, int rows, int hq,
                                       const int32_t* positions, const int32_t* counts, const float* inv_freq,
                                       const mt_kv8_cache* cache, float* q_out, int ldqo) {
    const char* what = "mt_rope_cache_kv8";
    MT_REQUIRE(ctx, qkv && positions && inv_freq && q_out, MT_ERR_ARG, "%s: null argument", what);
    mt_status st = kv8_check_cache(ctx, what, cache, requests);
    if (st != MT_OK) return st;
    const int hkv = cache->kv_heads;
    st = kv8_check_rows(ctx, what, requests, rows, hq, hkv);
    if (st != MT_OK) return st;
    MT_REQUIRE(ctx, ldq >= (hq + 2 * hkv) * 64 && ldqo >= hq * 64 && (q_out != qkv || ldqo == ldq), MT_ERR_SHAPE,
               "%s: hq %d hkv %d ldq %d ldqo %d", what, hq, hkv, ldq, ldqo);
    MT_REQUIRE(ctx, rows <= cache->capacity, MT_ERR_CAPACITY, "%s: %d rows exceed capacity %d", what, rows, cache->capacity);
    MT_REQUIRE(ctx, ctx, MT_ERR_ARG, "%s: null context", what);
    if (requests == 0 || rows == 0) return MT_OK;
    DeviceGuard guard(ctx->device);
    MT_REQUIRE(ctx, guard.err == cudaSuccess, MT_ERR_CUDA, "%s: %s", what, cudaGetErrorString(guard.err));
    AppendArgs a{};
    a.qkv = qkv; a.ldq = ldq; a.q_out = q_out; a.ldqo = ldqo;
    a.rows = Kv8Rows{positions, counts, rows, cache->base};
    a.total = requests * rows; a.hq = hq; a.hkv = hkv;
    // One row a block until the rows are two waves of blocks: a decode step is bound by its latency.
    const int per_sm = (a.total + 2 * ctx->sm_count - 1) / (2 * ctx->sm_count);
    a.block_rows = per_sm < AP_MAX_ROWS ? per_sm : AP_MAX_ROWS;
    a.vec = (((uintptr_t)qkv | (uintptr_t)q_out) & 15u) == 0 && ldq % 4 == 0 && ldqo % 4 == 0;
    a.inv_freq = inv_freq;
    a.k = cache->k; a.v = cache->v; a.k_scale = cache->k_scale; a.v_scale = cache->v_scale;
    a.request_stride = cache->request_stride; a.capacity = cache->capacity;
    const int blocks = (a.total + a.block_rows - 1) / a.block_rows;
    launch_k(cache->kind == MT_KV_INT8 ? rope_cache_kv8_kernel<MT_KV_INT8> : rope_cache_kv8_kernel<MT_KV_E4M3>, blocks,
             AP_THREADS, 0, as_stream(stream), a);
    return check_launch(ctx, what);
}

extern "C" mt_status mt_kv8_read(mt_ctx* ctx, void* stream, const mt_kv8_cache* cache, int requests, int rows,
                                 const int32_t* positions, const int32_t* counts, float* k, float* v, int out_capacity) {
    const char* what = "mt_kv8_read";
    MT_REQUIRE(ctx, positions && (k || v), MT_ERR_ARG, "%s: null argument", what);
    mt_status st = kv8_check_cache(ctx, what, cache, requests);
    if (st != MT_OK) return st;
    const int hkv = cache->kv_heads;
    st = kv8_check_rows(ctx, what, requests, rows, hkv, hkv);
    if (st != MT_OK) return st;
    MT_REQUIRE(ctx, rows <= cache->capacity && rows <= out_capacity, MT_ERR_CAPACITY,
               "%s: %d rows exceed capacity %d or out_capacity %d", what, rows, cache->capacity, out_capacity);
    MT_REQUIRE(ctx, (((uintptr_t)k | (uintptr_t)v) & 15u) == 0, MT_ERR_ARG, "%s: k and v need 16-byte alignment", what);
    MT_REQUIRE(ctx, ctx, MT_ERR_ARG, "%s: null context", what);
    if (requests == 0 || rows == 0) return MT_OK;
    DeviceGuard guard(ctx->device);
    MT_REQUIRE(ctx, guard.err == cudaSuccess, MT_ERR_CUDA, "%s: %s", what, cudaGetErrorString(guard.err));
    ReadArgs a{};
    a.rows = Kv8Rows{positions, counts, rows, cache->base};
    a.hkv = hkv; a.capacity = cache->capacity; a.out_capacity = out_capacity; a.request_stride = cache->request_stride;
    a.tiles = (rows + RD_ROWS - 1) / RD_ROWS;
    a.codes[0] = cache->k; a.codes[1] = cache->v; a.scale[0] = cache->k_scale; a.scale[1] = cache->v_scale;
    a.out[0] = k; a.out[1] = v;
    const long long blocks = (long long)a.tiles * hkv * requests;
    MT_REQUIRE(ctx, blocks <= 0x7FFFFFFFll, MT_ERR_SHAPE, "%s: %d requests of %d rows", what, requests, rows);
    launch_k(cache->kind == MT_KV_INT8 ? kv8_read_kernel<MT_KV_INT8> : kv8_read_kernel<MT_KV_E4M3>, (unsigned)blocks,
             RD_THREADS, 0, as_stream(stream), a);
    return check_launch(ctx, what);
}
