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
constexpr int AP_HEADS = 4;     // query heads of a group in flight (of 14, when 8 rows leave a row 4 groups)

struct AppendArgs {
    const float* qkv; int ldq;
    float* q_out; int ldqo;
    Kv8Rows rows;
    int total;           // requests * rows
    int hq, hkv;
    int block_rows;      // rows per block, <= AP_MAX_ROWS
    int parts;           // groups of 8 lanes per row
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

// Codes of four values: x / scale, whose exact quotient is rounded once, to the nearest code, ties to
// even. The product with the rounded reciprocal is off by a unit or two of fp32, which only matters
// next to a border between two codes; the remainder there, from one multiply-add, is exact and decides.
// int8: c is the nearest whole number (the sum with 1.5 * 2^23 has it in its low bits) or its neighbour,
//   and d = x - c scale is a multiple of half a unit of scale below 2^24 of them. 2|d| against scale says
//   whether c has to take a step towards x; at a tie an odd c takes it.
// e4m3: t is the quotient to 12 bits. Codes and borders between them have 5 bits or fewer, so where the
//   quotient is next to one, t is that one; d = x - t scale has the exact sign of the difference, and t
//   moves by its own last bit to that side. The conversion cannot be caught on a tie after that.
// Scales below 2^-60 are taken 2^64 higher, with x, so that no d is lost below the smallest number.
template <int KIND>
__device__ __forceinline__ uint32_t encode4(float4 x4, float scale, float rcp) {
    const float x[4] = {x4.x, x4.y, x4.z, x4.w};
    uint32_t code[4];
    if constexpr (KIND == MT_KV_INT8) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float m = fmaf(x[i], rcp, 12582912.f), c = m - 12582912.f;
            const float d = fmaf(-c, scale, x[i]), twice = fabsf(d) + fabsf(d);
            const uint32_t u = __float_as_uint(m);
            const bool step = twice > scale || (twice == scale && (u & 1u));
            code[i] = step ? u + (d < 0.f ? ~0u : 1u) : u;
        }
        return __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t t = (__float_as_uint(x[i] * rcp) + 0x800u) & 0xFFFFF000u;
            const float d = fmaf(-__uint_as_float(t), scale, x[i]);
            const uint32_t away = (uint32_t)((int)(__float_as_uint(d) ^ t) >> 31) | 1u;  // 1: |x / scale| > |t|, else -1
            code[i] = d == 0.f ? t : t + away;
        }
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(code[0]), __uint_as_float(code[1])), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(code[2]), __uint_as_float(code[3])), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}

// RoPE, quantisation and the cache write. A block takes block_rows rows; 8 lanes are a group, which has
// one row and every parts-th of its heads; lane j has the pairs (4j .. 4j+3, +32), so that loads and
// stores of a head are whole 128-byte lines and a code row is 16 words. The angles are made in 64 bits,
// one thread each (a position of 10^5 leaves an fp32 angle with 2 digits less, and a code is the same for
// every caller only if the rotated key is: rounding it once from 64 bits makes it so), while the loads of
// the group's first heads are under way. Queries are not quantised, and are turned in 32 bits with cosines and sines
// rounded once from 64: 3.6e-8 off in the mean instead of one rounding's 2.5e-8, a tenth of what attention adds.
// A decode step is bounded by its launch (2.7 us for 1 to 64 requests of 14 + 2 + 2 heads), prompts by latency (memory
// and 64-bit angles, 49% of the issue slots used): 4128 rows in 8.6 us, 4.0 TB/s; 1764 instructions a row before
// angles, divisions and conversions were shared out as here, 1000 now.
template <int KIND>
__global__ void __launch_bounds__(AP_THREADS, 3) rope_cache_kv8_kernel(const AppendArgs a) {
    __shared__ __align__(16) double turn[AP_MAX_ROWS][2][32];  // cos, sin
    __shared__ __align__(16) float turn_f[AP_MAX_ROWS][2][32];
    const int j = threadIdx.x & 7, group = threadIdx.x >> 3;
    const int row0 = blockIdx.x * a.block_rows;
    const int n = min(a.block_rows, a.total - row0);
    const int i = group / a.parts, part = group - i * a.parts;
    const int request = (row0 + i) / a.rows.rows, at = (row0 + i) - request * a.rows.rows;
    pdl_wait();
    pdl_launch();
    const Kv8Span s = kv8_span(a.rows, i < n ? request : 0);
    const bool on = i < n && at < s.count;
    const float* src = a.qkv + (size_t)(row0 + i) * a.ldq + 4 * j;
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    auto load = [&](float4 (&x)[2], int head, int end) {
        const bool here = on && head < end;
        x[0] = here ? load4(src + (size_t)head * 64, a.vec) : none;
        x[1] = here ? load4(src + (size_t)head * 64 + 32, a.vec) : none;
    };
    float4 c[2], q[AP_HEADS][2];
    load(c, a.hq + part, a.hq + 2 * a.hkv);
#pragma unroll
    for (int h = 0; h < AP_HEADS; h++) load(q[h], part + h * a.parts, a.hq);

    {
        const int row = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int request_r = (row0 + row) / a.rows.rows, at_r = (row0 + row) - request_r * a.rows.rows;
        if (row < n) {
            const Kv8Span r = kv8_span(a.rows, request_r);
            if (at_r < r.count) {
                double sn, cs;
                sincos((double)(r.pos + at_r) * (double)a.inv_freq[lane], &sn, &cs);
                turn[row][0][lane] = cs;
                turn[row][1][lane] = sn;
                turn_f[row][0][lane] = (float)cs;
                turn_f[row][1][lane] = (float)sn;
            }
        }
    }
    __syncthreads();

    if (on) {
        const float4 cs = *reinterpret_cast<const float4*>(&turn_f[i][0][4 * j]);
        const float4 sn = *reinterpret_cast<const float4*>(&turn_f[i][1][4 * j]);
        float* dst = a.q_out + (size_t)(row0 + i) * a.ldqo + 4 * j;
        for (int h0 = part; h0 < a.hq; h0 += AP_HEADS * a.parts) {
#pragma unroll
            for (int h = 0; h < AP_HEADS; h++) {
                const int head = h0 + h * a.parts;
                if (head >= a.hq) break;
                const float4 x = q[h][0], y = q[h][1];
                store4(dst + (size_t)head * 64, make_float4(x.x * cs.x - y.x * sn.x, x.y * cs.y - y.y * sn.y,
                                                            x.z * cs.z - y.z * sn.z, x.w * cs.w - y.w * sn.w), a.vec);
                store4(dst + (size_t)head * 64 + 32, make_float4(y.x * cs.x + x.x * sn.x, y.y * cs.y + x.y * sn.y,
                                                                 y.z * cs.z + x.z * sn.z, y.w * cs.w + x.w * sn.w), a.vec);
            }
            if (h0 + AP_HEADS * a.parts < a.hq) {
#pragma unroll
                for (int h = 0; h < AP_HEADS; h++) load(q[h], h0 + (AP_HEADS + h) * a.parts, a.hq);
            }
        }
    }
    // Whole warps run every iteration (the scale is a maximum over 8 lanes).
    const int slot = on ? (s.pos + at - a.rows.base) % a.capacity : 0;
    for (int u0 = 0; u0 < 2 * a.hkv; u0 += a.parts) {
        const int unit = u0 + part;
        const bool here = on && unit < 2 * a.hkv, value = unit >= a.hkv;
        if (u0 > 0) load(c, a.hq + unit, a.hq + 2 * a.hkv);
        float4 x = c[0], y = c[1];
        if (here && !value) {
            const double2* cs = reinterpret_cast<const double2*>(&turn[i][0][4 * j]);
            const double2* sn = reinterpret_cast<const double2*>(&turn[i][1][4 * j]);
            const double2 c0 = cs[0], c1 = cs[1], s0 = sn[0], s1 = sn[1];
            auto rot = [](float& p, float& q, double c, double s) {
                const double pd = p, qd = q;
                p = (float)(pd * c - qd * s);
                q = (float)(qd * c + pd * s);
            };
            rot(x.x, y.x, c0.x, s0.x); rot(x.y, y.y, c0.y, s0.y);
            rot(x.z, y.z, c1.x, s1.x); rot(x.w, y.w, c1.y, s1.y);
        }
        // max|x| over the head's 8 lanes as bit patterns: those of NaN and infinity are the largest.
        const float m0 = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        const float m1 = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
        const float sum = fabsf(x.x) + fabsf(x.y) + fabsf(x.z) + fabsf(x.w) + fabsf(y.x) + fabsf(y.y) + fabsf(y.z) +
                          fabsf(y.w);  // NaN if any is (fmaxf drops NaN)
        uint32_t top = sum != sum ? 0x7FFFFFFFu : __float_as_uint(fmaxf(m0, m1));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (!here) continue;
        const size_t to = (size_t)request * a.request_stride + (size_t)(value ? unit - a.hkv : unit) * a.capacity + slot;
        float scale = __fdiv_rn(__uint_as_float(top), KIND == MT_KV_INT8 ? 127.f : 448.f);
        uint32_t w0 = 0, w1 = 0;
        if (top >= 0x7F800000u) {
            scale = __uint_as_float(0x7FC00000u);
        } else if (scale < 1.17549435e-38f) {
            scale = 0.f;
        } else {
            float by = scale;
            if (scale < 8.67361738e-19f) {  // 2^-60
                const float up = 1.8446744e19f;  // 2^64
                by *= up;
                x.x *= up; x.y *= up; x.z *= up; x.w *= up;
                y.x *= up; y.y *= up; y.z *= up; y.w *= up;
            }
            const float rcp = __fdiv_rn(1.f, by);
            w0 = encode4<KIND>(x, by, rcp);
            w1 = encode4<KIND>(y, by, rcp);
        }
        uint32_t* codes = reinterpret_cast<uint32_t*>((value ? a.v : a.k) + to * 64);
        codes[j] = w0;
        codes[8 + j] = w1;
        if (j == 0) (value ? a.v_scale : a.k_scale)[to] = scale;
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
// Bounded by the fp32 stores: 64 requests of up to 500 rows in 6.0 us, 3.4 TB/s with the launch. The eight loads
// of a thread (four rows of keys, four of values) are issued before the first is used.
template <int KIND>
__global__ void __launch_bounds__(RD_THREADS) kv8_read_kernel(ReadArgs a) {
    const int tile = blockIdx.x % a.tiles, unit = blockIdx.x / a.tiles;
    const int head = unit % a.hkv, request = unit / a.hkv;
    pdl_wait();
    pdl_launch();
    const Kv8Span s = kv8_span(a.rows, request);
    const int lane = threadIdx.x & 15;
    const size_t from = (size_t)request * a.request_stride + (size_t)head * a.capacity;
    const int start = s.count > 0 ? (s.pos - a.rows.base) % a.capacity : 0;
    uint32_t w[2][RD_ROWS / 16];
    float sc[2][RD_ROWS / 16];
#pragma unroll
    for (int i = 0; i < RD_ROWS / 16; i++) {
        const int row = tile * RD_ROWS + i * 16 + (threadIdx.x >> 4);
        const int slot = row < s.count ? start + row : 0;  // row < capacity
        const size_t at = from + (slot >= a.capacity ? slot - a.capacity : slot);
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
                const uint32_t u = c ^ 0x80808080u;  // code + 128, the low byte of 2^23 + 128 + code
                auto code = [u](uint32_t byte) { return __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540u | byte)) - 8388736.f; };
                x = make_float4(code(0), code(1), code(2), code(3));
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
    const int per_sm = (a.total - 1) / (2 * ctx->sm_count) + 1;
    a.block_rows = per_sm < AP_MAX_ROWS ? per_sm : AP_MAX_ROWS;
    a.parts = AP_THREADS / 8 / a.block_rows;
    a.vec = (((uintptr_t)qkv | (uintptr_t)q_out) & 15u) == 0 && ldq % 4 == 0 && ldqo % 4 == 0;
    a.inv_freq = inv_freq;
    a.k = cache->k; a.v = cache->v; a.k_scale = cache->k_scale; a.v_scale = cache->v_scale;
    a.request_stride = cache->request_stride; a.capacity = cache->capacity;
    const int blocks = (a.total - 1) / a.block_rows + 1;
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
