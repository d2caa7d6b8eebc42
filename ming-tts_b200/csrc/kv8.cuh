// kv8.cuh -- shared by the 8-bit key/value cache kernels (kv8.cu, kv8_attention.cu).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace mt {

// A request's rows, read by every kernel of a call: its first position and how many rows are its own
// (0 for an idle request: a position below `base`, or positions that would pass 2^31 - 1).
struct Kv8Rows {
    const int* positions;
    const int* counts;  // optional
    int rows, base;
};
struct Kv8Span {
    int pos, count;
};
__device__ __forceinline__ Kv8Span kv8_span(const Kv8Rows& a, int request) {
    Kv8Span s;
    s.pos = a.positions[request];
    s.count = a.counts ? min(max(a.counts[request], 0), a.rows) : a.rows;
    if (s.pos < a.base || s.pos > 0x7FFFFFFF - a.rows) s.count = 0;
    return s;
}

// Host-side checks that the entry points share. `what` names the entry point.
mt_status kv8_check_cache(mt_ctx* ctx, const char* what, const mt_kv8_cache* c, int requests);
mt_status kv8_check_rows(mt_ctx* ctx, const char* what, int requests, int rows, int hq, int hkv);

// ------------------------------------------------------------------------------------------------
// Attention (kv8_attention.cu, kv8_attention_wide.cu)
// ------------------------------------------------------------------------------------------------
struct Kv8View {
    const uint8_t *k, *v;
    const float *ks, *vs;
    long long request_stride;
    int capacity, kind;
};

// One pass over one set of keys: a request's own cache (units: request x kv head, causal), or the
// shared prefix (units: kv heads, the rows of all requests in one tile space, every key seen).
struct PassArgs {
    const float* q; int ldq; bool qvec;
    float* out; int ldo; bool ovec;  // written when the pass has one part
    Kv8Rows rows;
    int requests, hq, hkv, group, window;
    Kv8View c;
    int prefix_len;                  // > 0: the prefix pass
    int units, row_blocks, splits;   // grid: units (pack of them a block) x row_blocks x splits, or
    int pack, unit_tiles;            // units with fewer row tiles (unit_tiles) than a block has room for share it
    int slots;                       // > 0: slots x kv heads x row_blocks, the slots shared out by length (kv8_share)
    int2* shares;                    // per request: its first slot and their number, for the join
    int key_warps;                   // warps of a block that share a row tile and interleave its keys
    bool parted;                     // the outputs go to parts, for the join: 64 sums, and (reference, sum of weights)
    float *part_o, *part_ml;         // [row * hq + head][splits], or request by request [pair][its slots]
    size_t part0;                    // this pass's first
    // The pass before this one in the stream is the same call's other pass: they write different parts, so
    // this one runs beside it and waits for it at its end (every block of that pass has waited for what
    // came before the call, or this one would not have been launched).
    bool beside;
};

// Begins a pass. Beside another, what the kernels before the call wrote is complete and in L2; the fence is
// there for lines of it that this SM's L1 may still hold from an earlier step.
__device__ __forceinline__ void pass_begin(bool beside) {
    if (beside) asm volatile("fence.acq_rel.gpu;" ::: "memory");
    else pdl_wait();
    pdl_launch();
}

// Where the keys of a tile of rows are. Index u counts positions from a multiple of the capacity, so that
// slot(u) is u or u - capacity; the tile's rows see [lo, hi] at most, and all of [in_lo, in_hi].
struct KeyRange {
    size_t row;  // first slot of the request and head
    int lo, hi, in_lo, in_hi, capacity;
    __device__ __forceinline__ size_t slot(int u) const {  // u outside the range: the nearest inside it
        u = min(max(u, lo), hi);
        return row + (u >= capacity ? u - capacity : u);
    }
    // Slots u0 .. u0 + n - 1 are in the range and side by side.
    __device__ __forceinline__ bool whole(int u0, int n) const {
        return u0 >= lo && u0 + n - 1 <= hi && (u0 + n <= capacity || u0 >= capacity);
    }
};

// A unit's row space: rows x group (row, head) pairs, row-major. In a pass over a request's own cache a
// unit is (request, kv head), in a prefix pass a kv head and the rows are those of all requests.
struct UnitRows {
    const PassArgs& a;
    int request, kvh;
    Kv8Span span;  // of the request
    int first;     // oldest position that the cache holds
    int shift;     // position of u = 0
    KeyRange keys;

    __device__ __forceinline__ UnitRows(const PassArgs& args, int unit) : a(args) {
        const bool prefix = a.prefix_len > 0;
        request = prefix ? 0 : unit / a.hkv;
        kvh = prefix ? unit : unit % a.hkv;
        keys.capacity = a.c.capacity;
        keys.row = (size_t)request * a.c.request_stride + (size_t)kvh * a.c.capacity;
        shift = 0;
    }
    // Reads the request's span: the rest needs it.
    __device__ __forceinline__ void locate() {
        if (a.prefix_len > 0) return;
        span = kv8_span(a.rows, request);
        first = max(a.rows.base, span.pos + span.count - a.c.capacity);
    }
    // (row, head) pairs of the unit.
    __device__ __forceinline__ int size() const {
        return (a.prefix_len > 0 ? a.requests * a.rows.rows : span.count) * a.group;
    }
    // Sets `keys` for the pairs e0 .. e0 + n - 1 (e0 < size()).
    __device__ __forceinline__ void tile(int e0, int n) {
        if (a.prefix_len > 0) {
            keys.lo = 0; keys.hi = a.prefix_len - 1; keys.in_lo = 0; keys.in_hi = keys.hi;
            return;
        }
        const int i0 = e0 / a.group, i1 = min((e0 + n - 1) / a.group, span.count - 1);
        const int from = oldest(i0);
        shift = from - (from - a.rows.base) % a.c.capacity;
        keys.lo = from - shift;
        keys.hi = span.pos + i1 - shift;
        keys.in_lo = oldest(i1) - shift;
        keys.in_hi = span.pos + i0 - shift;
    }
    // Oldest position that row i sees.
    __device__ __forceinline__ int oldest(int i) const {
        return a.window > 0 ? max(first, span.pos + i - a.window + 1) : first;
    }
    // Pair e: row * hq + head, or -1 where it is not one of a request's own, and the keys [lo, hi] it sees.
    __device__ __forceinline__ int pair(int e, int& lo, int& hi) const {
        lo = keys.lo; hi = keys.hi;
        if (e >= size()) return -1;
        const int i = e / a.group, head = kvh * a.group + e - i * a.group;
        if (a.prefix_len > 0) {
            const int req = i / a.rows.rows;
            return i - req * a.rows.rows < kv8_span(a.rows, req).count ? i * a.hq + head : -1;
        }
        hi = span.pos + i - shift;
        lo = oldest(i) - shift;
        return (request * a.rows.rows + i) * a.hq + head;
    }
};

constexpr float KV8_REF_NONE = -3.4028235e38f;  // reference of a row that has seen no key: no score is below it

// The kernel for many rows (kv8_attention_wide.cu): blocks of KV8_WIDE_ROWS rows, `splits` parts of
// `chunk` tiles of KV8_WIDE_KEYS keys each.
constexpr int KV8_WIDE_ROWS = 256, KV8_WIDE_KEYS = 64;
void launch_kv8_wide(const PassArgs& a, int chunk, unsigned int* status, cudaStream_t s);

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float rcp(float x) {  // within one unit of the last place
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Codes of bytes 0, 1 and of bytes 2, 3 as two fp16 pairs. Integers: the byte with its sign bit
// flipped, put under fp16's 1024 (0x64), is 1024 + 128 + code.
template <int KIND>
__device__ __forceinline__ void to_half(uint32_t w, uint32_t& h01, uint32_t& h23) {
    if (KIND == MT_KV_INT8) {
        w ^= 0x80808080u;
        const uint32_t bias = 0x64806480u;  // 1152, 1152
        uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(h01) : "r"(a), "r"(bias));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(h23) : "r"(b), "r"(bias));
    } else {
        asm("{.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;}"
            : "=r"(h01), "=r"(h23)
            : "r"(w));
    }
}

// Two values as fp16 pairs hi + lo.
__device__ __forceinline__ void split_half2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 2^(target - e) for x in [2^e, 2^(e+1)), within 2^+-126.
__device__ __forceinline__ float power_to(float x, int target) {
    const int e = (int)(__float_as_uint(x) >> 23) - 127;
    return __uint_as_float((uint32_t)(min(126, max(-126, target - e)) + 127) << 23);
}

// The units of a row. Weights are 2^(score - off), off = reference - lift: the reference is near a score that was the
// row's largest. Products of a weight and its value scale go into the planes times `extra`, a power of two: lift and
// extra, 2^total together, bring the largest product to 1 when they are set. The two planes hold 22 bits of
// products down to 2^-3 of it, 2^-25 of it below, and have room for 2^15 above. How much of the total is lift is a
// kernel's own choice: a lift rounds the exponents of the largest weights to its own size, an extra that is a row's
// own takes a multiplication. A row moves its units only when a product leaves their room (or a weight fp32's):
// keeping the products near 2^8 instead moved it ten times as often, and cost 10% of the wide kernel's time.
constexpr float KV8_UNSET = 1000.f;           // the total of a row that has seen no value but zeros
constexpr float KV8_FAR = 400.f;              // in a total (between 200 and 600 then): the row has no lift, see kv8_move
constexpr float KV8_PRODUCT_MAX = 32768.f;    // fp16 ends at 65504
constexpr float KV8_WEIGHT_MAX = 0x1p100f;    // what a sum of four weights may be

__device__ __forceinline__ float kv8_power(float n) { return __uint_as_float((uint32_t)((int)n + 127) << 23); }  // 2^n, |n| <= 126

// A score in powers of two, rounded. off is taken from scores so rounded, and so are the weights of the keys that it
// is taken from: at 10^9 one multiply-add gives another score by up to 2^6, which is 2^64 in a weight.
__device__ __forceinline__ float kv8_score(float sum, float scale) { return __fmul_rn(sum, scale); }

// Sets off and total of a row after four of a lane's keys (scores z in powers of two, -infinity where not seen,
// value scales v), to the same in all four lanes of the row; lift(total) is the lift. Returns what the row's sum of
// weights and its outputs so far have to be multiplied by: neither grows, but for sums of a row without units.
// Where fp32 has no fraction at the reference (from 2^24 on) a lift would be rounded: extra takes all of the total.
struct Kv8Move {
    float sums, outputs;
};
template <typename Lift>
__device__ __forceinline__ Kv8Move kv8_move(const float (&z)[4], const float (&v)[4], float& off, float& total, Lift&& lift) {
    auto row_max = [](float x) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    };
    auto product = [&](float from) {  // the largest, in units of 2^from
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) x = fmaxf(x, ex2(z[j] - from) * v[j]);
        return row_max(x);
    };
    const bool unset = total == KV8_UNSET;
    const float most = row_max(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
    const bool was_far = !unset && total > 0.5f * KV8_FAR;
    const float old = was_far ? total - KV8_FAR : total;
    const float old_lift = unset || was_far ? 0.f : lift(old), old_extra = unset ? 0.f : old - old_lift;  // of 2
    const float now = __any_sync(0xffffffffu, !unset) ? product(off) * kv8_power(old_extra) : 0.f;
    const bool move = most > -INFINITY && (unset || most - off > 90.f || now > KV8_PRODUCT_MAX);
    const float ref = fmaxf(off + old_lift, most);
    const float then = product(ref);
    if (!move) return Kv8Move{1.f, 1.f};
    // No product but zeros yet: the weights have their unit, the products wait for theirs.
    const bool none = unset && then == 0.f;
    float to = then > 0.f ? fminf(126.f, fmaxf(-126.f, (float)(127 - (int)(__float_as_uint(then) >> 23)))) : old;
    if (!unset) to = fminf(to, old + floorf(ref - (off + old_lift)));  // what is there may be the larger part
    float new_lift = none ? 0.f : lift(to);
    const bool far = fabsf(ref) >= 0x1p24f && new_lift != 0.f;
    if (far) new_lift = 0.f;
    const float sums = ex2(off - (ref - new_lift));
    off = ref - new_lift;
    total = far ? to + KV8_FAR : to;
    return Kv8Move{sums, unset ? 0.f : sums * kv8_power(to - new_lift) * kv8_power(-old_extra)};
}

// A row's sum of weights, in units of 2^off, as (reference, sum) with sum in [1, 2): whatever its units,
// sums of several parts can be compared and added. The outputs that go with it are already divided by it,
// so that no step on the way is larger than the largest value, which may be near fp32's largest.
__device__ __forceinline__ float2 kv8_total(float off, float sum) {
    if (sum == 0.f) return make_float2(KV8_REF_NONE, 0.f);
    const float p = power_to(sum, 0);
    return make_float2(off + (float)(127 - (int)(__float_as_uint(p) >> 23)), sum * p);
}

// Outputs (times `extra`, a power of two) divided by the sum of weights: extra and the sum's power of two
// in two halves, the rest of the sum, in [1, 2), with the first. No product leaves fp32 where the result does not.
struct OverSum {
    float first, second;
    __device__ __forceinline__ OverSum(float extra, float sum) {
        const float p = power_to(sum, 0);
        const int e = (int)(__float_as_uint(p) >> 23) - (int)(__float_as_uint(extra) >> 23), half = e >> 1;
        first = sum == 0.f ? 0.f : __uint_as_float((uint32_t)(half + 127) << 23) * rcp(sum * p);
        second = __uint_as_float((uint32_t)(e - half + 127) << 23);
    }
    __device__ __forceinline__ float operator()(float x) const { return x * first * second; }
};

// Makes a device current for a call and puts the caller's back.
struct DeviceGuard {
    int before = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device)
            err = cudaSetDevice(device);
        else
            before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

}  // namespace mt
