// kv8_attention_wide.cu -- attention over an 8-bit cache for many rows (prompts, batches behind a shared
// prefix) on the tcgen05 tensor cores. The arithmetic is that of kv8_attention.cu: codes exact in fp16,
// queries and weights as two fp16 planes, fp32 sums.
//
// A block takes 256 (row, head) pairs of one kv head, as two tiles of 128, and walks its keys 64 at a
// time. Its warps:
//   0-3, 4-7  the rows of tile 0, 1: a thread a row. It reads the row's scores from TMEM, keeps the
//             reference and the sum, writes the weights (times the value rows' scales) back as two fp16
//             planes over the scores, and adds each key tile's output, read from TMEM, to 64 registers.
//   8-11      convert codes to fp16 in shared memory (four stages), K and V alike: a key a 128-byte row
//   12 (of the last four) issues the matrix instructions: S = Q K^T (128 x 64, both planes of Q from TMEM)
//             and O = P V (128 x 64, both planes of P from TMEM; V is the [key][dimension] tile as it is)
// The scores of the next key tile are in a second buffer while a tile's weights are made, so neither the
// row threads nor the tensor cores wait for the other in turn.
//
// Every key tile's O starts from zero: the accumulators drop the bits that 24 do not hold, and a chain of
// 64 keys keeps that near fp32's own rounding; it also leaves nothing in TMEM to rescale.
//
// TMEM, 256 columns a row tile: 0-63 and 64-127 scores of even and odd key tiles (fp32), overwritten 16
// columns at a time by 8 columns of hi and 8 of lo planes of the same 16 keys' weights; 128-191 the
// query planes in the same way; 192-255 O.
#include <math.h>

#include "kv8.cuh"

namespace mt {

namespace {

constexpr int WD_ROW_WARPS = 8, WD_CONVERT_WARPS = 4;
constexpr int WD_THREADS = 32 * (WD_ROW_WARPS + WD_CONVERT_WARPS + 4);
// Registers of a thread, by warpgroup: the block starts with 512 x 128 = 65,536 of them, and
// 256 x 168 + 128 x 96 + 128 x 80 is as many.
constexpr int WD_ROW_REGS = 168, WD_CONVERT_REGS = 96, WD_ISSUE_REGS = 80;
constexpr int WD_KEYS = KV8_WIDE_KEYS;
constexpr int WD_STAGE = WD_KEYS * 128;  // bytes of a K or V tile in fp16
constexpr int WD_STAGES = 4;
constexpr int WD_PLANE = 128 * 128;      // bytes of a plane of a tile's queries
constexpr size_t WD_SMEM = 2 * WD_STAGES * WD_STAGE + 4 * WD_PLANE + 1024;
constexpr uint32_t T_Q = 128, T_O = 192, T_TILE = 256;
constexpr float WD_LIFT_MAX = 118.f;  // largest power that the weights are scaled by
constexpr int WD_LIFT_TO = 8;         // exponent that a row's largest scaled product is brought to ..
constexpr float WD_PRODUCT_MAX = 32768.f;  // .. once one is above this (fp16 ends at 65504)
constexpr float WD_WEIGHT_MAX = 0x1p100f;

// 16 columns of this thread's lane: issue, and wait for every load issued so far (the registers are
// operands of the wait, so nothing uses them before it).
__device__ __forceinline__ void tmem_ld16(uint32_t at, float (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_ld_wait(float (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                   "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&u)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
        : "memory");
}

// Calls f(c, columns 16 c ..) for c = 0 .. N-1 with the next columns' load in flight.
template <int N, typename F>
__device__ __forceinline__ void tmem_walk(uint32_t at, F&& f) {
    float x[16], y[16];
    tmem_ld16(at, x);
#pragma unroll 1
    for (int c = 0; c < N; c += 2) {
        tmem_ld_wait(x);
        tmem_ld16(at + 16 * c + 16, y);
        f(c, x);
        tmem_ld_wait(y);
        if (c + 2 < N) tmem_ld16(at + 16 * c + 32, x);
        f(c + 1, y);
    }
}

// TMEM stores of this thread done and ordered before what another thread does after a barrier.
__device__ __forceinline__ void tmem_publish() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_acquire() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D[tmem] (+)= A[tmem] B[shared], fp16 operands, fp32 accumulator, M = 128.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// One thread of the warp, in a form that the compiler knows to be one: its matrix instructions then take
// their operands from uniform registers (an O step was 45 cycles behind `lane == 0`, 32 behind this).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_done(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// Descriptor of a tile of 128-byte rows in the 128-byte swizzle (16-byte chunk c of row r at chunk
// c ^ (r % 8); 8-row groups 1024 bytes apart): K with the contraction along the row (keys are rows of
// B), V with the contraction across rows. The tile is one swizzle span wide, so the stride between
// 8-row groups is the only one that either reading uses; both offset fields hold it.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(1024 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
constexpr uint32_t IDESC_S = 1u << 4 | (WD_KEYS / 8) << 17 | (128 / 16) << 24;
constexpr uint32_t IDESC_O = 1u << 4 | 1u << 16 | (64 / 8) << 17 | (128 / 16) << 24;  // B with N along its rows

struct Shared {
    alignas(16) float ks[WD_STAGES][WD_KEYS], vs[WD_STAGES][WD_KEYS];  // scales of the stages' keys (values': / unit)
    float k_top[WD_STAGES][WD_CONVERT_WARPS];                          // largest norm of a key, by converting warp
    float first[WD_CONVERT_WARPS];
    float unit;                                                        // power of two near the first value scales
    uint64_t k_full[WD_STAGES], k_free[WD_STAGES], v_full[WD_STAGES], v_free[WD_STAGES];
    uint64_t q_ready[2], s_ready[2][2], p_ready[2], o_ready[2];        // by row tile (and key tile parity)
    uint32_t tmem;
    int abort;
};

// Two fp32 values in one register pair and the instructions that work on both.
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void f2_parts(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// A row's state. Weights are 2^(score - off), off = reference - lift: the reference is near a score that
// was the row's largest, the lift brings the largest weight times value scale to 2^8, where the planes
// have 22 bits for weights down to 2^-20 of it.
struct RowState {
    float off, lift;
    F2 sum;
    float o[64];
    float carry;  // by which the output not yet added is to be scaled

    __device__ __forceinline__ void scale(float f) {
        sum = f2_mul(sum, f2(f, f));
        carry *= f;
#pragma unroll
        for (int j = 0; j < 64; j++) o[j] *= f;
    }
};

// The keys of a tile as a row's thread sees them.
struct TileKeys {
    const float *ks, *vs;
    int u0, lo, hi;  // of the first key; the row sees [lo, hi]
};

template <bool MASK>
__device__ __forceinline__ bool sees(const TileKeys& t, int key) {
    return !MASK || (t.u0 + key >= t.lo && t.u0 + key <= t.hi);
}

// First tile, and where the weights could pass fp32's range: sets the reference to the row's largest
// score of this tile, and the lift.
__device__ __noinline__ float2 row_reference(uint32_t tm, const TileKeys& t, float rs, float off, float lift) {
    float top = -INFINITY;
    tmem_walk<4>(tm, [&](int c, const float(&s)[16]) {
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (sees<true>(t, 16 * c + j)) top = fmaxf(top, s[j] * t.ks[16 * c + j] * rs);
    });
    float ref = off + lift;
    if (top > ref) ref = top;
    float product = 0.f;
    tmem_walk<4>(tm, [&](int c, const float(&s)[16]) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float w = ex2(fmaf(s[j] * t.ks[16 * c + j], rs, -ref)) * fabsf(t.vs[16 * c + j]);
            if (sees<true>(t, 16 * c + j)) product = fmaxf(product, w);
        }
    });
    if (product * ex2(lift) > WD_PRODUCT_MAX)
        lift = fminf((float)(WD_LIFT_TO + 127 - (int)(__float_as_uint(product) >> 23)), WD_LIFT_MAX);
    return make_float2(ref, lift);
}

// Products of the tile so far (planes of `chunks` times 16 keys) scaled by f.
__device__ __noinline__ void row_rescale(uint32_t tm, int chunks, float f) {
    for (int c = 0; c < chunks; c++) {
        float x[16];
        uint32_t planes[16];
        tmem_ld16(tm + 16 * c, x);
        tmem_ld_wait(x);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&x[j]));
            const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&x[8 + j]));
            split_half2((hi.x + lo.x) * f, (hi.y + lo.y) * f, planes[j], planes[8 + j]);
        }
        tmem_st16(tm + 16 * c, planes);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
}

// Weights of the row in this tile: 2^(score - off), summed, and times the value scales into the planes.
template <bool MASK>
__device__ __forceinline__ void row_weights(uint32_t tm, const TileKeys& t, float rs, RowState& row) {
    const F2 rs2 = f2(rs, rs), minus = f2(-1.f, -1.f);
    tmem_walk<4>(tm, [&](int c, const float(&s)[16]) {
        const F2 off2 = f2(-row.off, -row.off);
        F2 w[8];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const ulonglong2 k4 = *reinterpret_cast<const ulonglong2*>(t.ks + 16 * c + j);
            const ulonglong2 v4 = *reinterpret_cast<const ulonglong2*>(t.vs + 16 * c + j);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const F2 k{i ? k4.y : k4.x}, v{i ? v4.y : v4.x};
                const bool on0 = sees<MASK>(t, 16 * c + j + i), on1 = sees<MASK>(t, 16 * c + j + i + 1);
                float x0, x1;
                f2_parts(f2_fma(f2_mul(f2(s[j + i], s[j + i + 1]), k), rs2, off2), x0, x1);
                const F2 p = f2(on0 ? ex2(x0) : 0.f, on1 ? ex2(x1) : 0.f);
                row.sum = f2_add(row.sum, p);
                w[(j + i) / 2] = f2_mul(p, v);
                f2_parts(w[(j + i) / 2], x0, x1);
                if (MASK) {  // a scale of a key that this row does not see may be NaN
                    x0 = on0 ? x0 : 0.f;
                    x1 = on1 ? x1 : 0.f;
                    w[(j + i) / 2] = f2(x0, x1);
                }
                top = fmaxf(top, fmaxf(fabsf(x0), fabsf(x1)));
            }
        }
        if (__any_sync(0xffffffffu, top > WD_PRODUCT_MAX)) {  // rare: the row's scale moves within the tile
            float f = 1.f;
            if (top > WD_PRODUCT_MAX && top <= 3.4e38f) {
                const int down = (int)(__float_as_uint(top) >> 23) - 127 - WD_LIFT_TO;
                f = __uint_as_float((uint32_t)(127 - min(down, 126)) << 23);
                row.off += (float)min(down, 126);
                row.lift -= (float)min(down, 126);
                row.scale(f);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            row_rescale(tm, c, f);
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = f2_mul(w[j], f2(f, f));
        }
        uint32_t planes[16];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x0, x1;
            f2_parts(w[j], x0, x1);
            const __half2 hi = __floats2half2_rn(x0, x1);
            const float2 back = __half22float2(hi);
            f2_parts(f2_fma(f2(back.x, back.y), minus, w[j]), x0, x1);
            const __half2 lo = __floats2half2_rn(x0, x1);
            planes[j] = *reinterpret_cast<const uint32_t*>(&hi);
            planes[8 + j] = *reinterpret_cast<const uint32_t*>(&lo);
        }
        tmem_st16(tm + 16 * c, planes);
    });
}

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int KIND>
__global__ void __launch_bounds__(WD_THREADS, 1) kv8_wide_kernel(const PassArgs a, int chunk, unsigned int* status) {
    extern __shared__ uint8_t dynamic[];
    __shared__ Shared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch();
    // Blocks with the most keys (the last rows) first.
    const int split = blockIdx.x % a.splits;
    const int unit = (blockIdx.x / a.splits) % a.units;
    const int row_block = a.row_blocks - 1 - blockIdx.x / (a.splits * a.units);
    UnitRows rows(a, unit);
    const int e0 = row_block * KV8_WIDE_ROWS, left = rows.size() - e0;
    if (left <= 0) return;
    rows.tile(e0, KV8_WIDE_ROWS);
    const KeyRange& r = rows.keys;
    const int u_first = (r.lo & ~15) + split * chunk * WD_KEYS;
    const int tiles = min(chunk, (r.hi - u_first) / WD_KEYS + 1);  // of this part
    if (u_first > r.hi) {
        if (warp < WD_ROW_WARPS) {
            int lo, hi;
            const int target = rows.pair(e0 + threadIdx.x, lo, hi);
            if (target >= 0)
                reinterpret_cast<float2*>(a.part_ml)[(size_t)target * a.parts + a.part0 + split] = make_float2(KV8_REF_NONE, 0.f);
        }
        return;
    }
    const int row_tiles = left > 128 ? 2 : 1;

    uint8_t* const stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dynamic) + 1023) & ~uintptr_t(1023));
    if (threadIdx.x == 0) {
        for (int i = 0; i < WD_STAGES; i++) {
            mbar_init(&sh.k_full[i], WD_CONVERT_WARPS);
            mbar_init(&sh.v_full[i], WD_CONVERT_WARPS);
            mbar_init(&sh.k_free[i], 1);
            mbar_init(&sh.v_free[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_ready[i], 4);
            mbar_init(&sh.s_ready[i][0], 1);
            mbar_init(&sh.s_ready[i][1], 1);
            mbar_init(&sh.p_ready[i], 4);
            mbar_init(&sh.o_ready[i], 1);
        }
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == WD_ROW_WARPS + WD_CONVERT_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    tmem_acquire();
    const uint32_t tmem = sh.tmem;
    volatile int* const abort = &sh.abort;

    if (warp < WD_ROW_WARPS) {
        more_registers<WD_ROW_REGS>();
        const int tile = warp >> 2;
        if (tile < row_tiles) {
            int lo, hi;
            const int target = rows.pair(e0 + threadIdx.x, lo, hi);
            const uint32_t tm = tmem + tile * T_TILE + ((uint32_t)(warp & 3) << 21);  // lanes 32 (warp % 4) ..
            float rs = 0.f;     // scores in powers of two: TMEM value x key scale x rs
            float reach = 0.f;  // no score is above reach x the key's norm
            {
                // Queries: four lanes a row, 16 dimensions each, 8 rows a pass.
                long long src = -1;
                if (target >= 0) {
                    const int row = target / a.hq;
                    src = (long long)row * a.ldq + (long long)(target - row * a.hq) * 64;
                }
                const int part = lane & 3;
                float x[4][16];
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const long long from = __shfl_sync(0xffffffffu, src, 8 * n + (lane >> 2));
                    const float* f = a.q + from + 16 * part;
                    if (from < 0) {
#pragma unroll
                        for (int j = 0; j < 16; j++) x[n][j] = 0.f;
                    } else if (a.qvec) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float4 y = reinterpret_cast<const float4*>(f)[j];
                            x[n][4 * j] = y.x; x[n][4 * j + 1] = y.y; x[n][4 * j + 2] = y.z; x[n][4 * j + 3] = y.w;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) x[n][j] = f[j];
                    }
                }
                uint8_t* const planes = stages + 2 * WD_STAGES * WD_STAGE + 2 * tile * WD_PLANE;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    float top = 0.f, norm = 0.f;
#pragma unroll
                    for (int j = 0; j < 16; j++) top = fmaxf(top, fabsf(x[n][j]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float up = power_to(top, 13);
                    const int row = 32 * (warp & 3) + 8 * n + (lane >> 2);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t qh[4], ql[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float y0 = x[n][8 * h + 2 * j] * up, y1 = x[n][8 * h + 2 * j + 1] * up;
                            norm = fmaf(y0, y0, fmaf(y1, y1, norm));
                            split_half2(y0, y1, qh[j], ql[j]);
                        }
                        const int at = row * 128 + (((2 * part + h) ^ (row & 7)) << 4);
                        *reinterpret_cast<uint4*>(planes + at) = make_uint4(qh[0], qh[1], qh[2], qh[3]);
                        *reinterpret_cast<uint4*>(planes + WD_PLANE + at) = make_uint4(ql[0], ql[1], ql[2], ql[3]);
                    }
                    norm += __shfl_xor_sync(0xffffffffu, norm, 1);
                    norm += __shfl_xor_sync(0xffffffffu, norm, 2);
                    const float r0 = __shfl_sync(0xffffffffu, 0.125f * 1.4426950408889634f / up, 4 * (lane & 7));
                    const float n0 = __shfl_sync(0xffffffffu, norm, 4 * (lane & 7));
                    if (lane >> 3 == n) {
                        rs = r0;
                        reach = 1.001f * sqrtf(n0) * r0;
                    }
                }
            }
            __syncwarp();
            {
                const int row = threadIdx.x & 127;
                const uint8_t* const planes = stages + 2 * WD_STAGES * WD_STAGE + 2 * tile * WD_PLANE + row * 128;
#pragma unroll
                for (int c = 0; c < 4; c++) {  // 16 dimensions: 8 columns of hi and 8 of lo
                    uint32_t x[16];
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const uint4 y = *reinterpret_cast<const uint4*>(planes + (h >> 1) * WD_PLANE + (((2 * c + (h & 1)) ^ (row & 7)) << 4));
                        x[4 * h] = y.x; x[4 * h + 1] = y.y; x[4 * h + 2] = y.z; x[4 * h + 3] = y.w;
                    }
                    tmem_st16(tm + T_Q + 16 * c, x);
                }
            }
            tmem_publish();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_ready[tile]);

            RowState row;
            row.off = KV8_REF_NONE; row.lift = WD_LIFT_MAX; row.carry = 1.f;
            row.sum = f2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 64; j++) row.o[j] = 0.f;
            auto add_output = [&]() {
                const F2 carry = f2(row.carry, row.carry);
                float y[2][16];
                tmem_ld16(tm + T_O, y[0]);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    tmem_ld_wait(y[c & 1]);
                    if (c < 3) tmem_ld16(tm + T_O + 16 * (c + 1), y[(c + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        float* o = row.o + 16 * c + j;
                        f2_parts(f2_fma(f2(y[c & 1][j], y[c & 1][j + 1]), carry, f2(o[0], o[1])), o[0], o[1]);
                    }
                }
            };
            bool ok = true;
            for (int n = 0; n < tiles; n++) {
                const int st = n & (WD_STAGES - 1), u0 = u_first + n * WD_KEYS;
                ok = mbar_wait(&sh.v_full[st], (n / WD_STAGES) & 1, status, 21, abort) &&  // the scales come with the values
                     mbar_wait(&sh.s_ready[tile][n & 1], (n >> 1) & 1, status, 20, abort);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tmem_acquire();
                const TileKeys keys{sh.ks[st], sh.vs[st], u0, lo, hi};
                const uint32_t tp = tm + (n & 1) * WD_KEYS;
                const float k_top = fmaxf(fmaxf(sh.k_top[st][0], sh.k_top[st][1]), fmaxf(sh.k_top[st][2], sh.k_top[st][3]));
                // |q.k| <= |q| |k|: no weight passes 2^100.
                if (__any_sync(0xffffffffu, !(ex2(reach * k_top - row.off) <= WD_WEIGHT_MAX))) {
                    const float2 rl = row_reference(tp, keys, rs, row.off, row.lift);
                    const float to = rl.x - rl.y;
                    if (to != row.off) row.scale(ex2(row.off - to));
                    row.off = to;
                    row.lift = rl.y;
                }
                if (u0 >= r.in_lo && u0 + WD_KEYS - 1 <= r.in_hi) row_weights<false>(tp, keys, rs, row);
                else row_weights<true>(tp, keys, rs, row);
                if (n > 0) {  // the last tile's output, before the next is written over it
                    ok = mbar_wait(&sh.o_ready[tile], (n - 1) & 1, status, 22, abort);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tmem_acquire();
                    add_output();
                }
                row.carry = 1.f;
                tmem_publish();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[tile]);
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_ready[tile], (tiles - 1) & 1, status, 22, abort));
            if (ok) {
                tmem_acquire();
                add_output();
                if (target >= 0) {
                    float s0, s1;
                    f2_parts(row.sum, s0, s1);
                    const float down = ex2(-row.lift), total = (s0 + s1) * down;
                    float f = sh.unit * down;
                    float* dst;
                    bool vec = true;
                    if (a.parts == 1) {
                        const int at = target / a.hq, head = target - at * a.hq;
                        dst = a.out + (size_t)at * a.ldo + (size_t)head * 64;
                        vec = a.ovec;
                        f /= total;
                    } else {
                        const size_t part = (size_t)target * a.parts + a.part0 + split;
                        reinterpret_cast<float2*>(a.part_ml)[part] = make_float2(row.off + row.lift, total);
                        dst = a.part_o + part * 64;
                    }
                    if (vec) {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            reinterpret_cast<float4*>(dst)[j] =
                                make_float4(row.o[4 * j] * f, row.o[4 * j + 1] * f, row.o[4 * j + 2] * f, row.o[4 * j + 3] * f);
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; j++) dst[j] = row.o[j] * f;
                    }
                }
            }
        }
    } else if (warp < WD_ROW_WARPS + WD_CONVERT_WARPS) {
        fewer_registers<WD_CONVERT_REGS>();
        // Four lanes a key, 16 codes each: 32 keys a pass. The next tile's codes are in registers while
        // this one's stage is waited for.
        const int i = threadIdx.x - 32 * WD_ROW_WARPS, part = i & 3, w = warp - WD_ROW_WARPS;
        uint4 k[2], v[2];
        float kn[2], ks = 0.f, vs = 0.f;  // scales of the keys whose codes this lane has; of key i
        auto load = [&](int u0) {
            const bool whole = r.whole(u0, WD_KEYS);
            const size_t at = r.row + (u0 >= r.capacity ? u0 - r.capacity : u0);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                // Keys outside the range stand in as the nearest inside it: see kv8_attention.cu.
                const int key = 32 * j + (i >> 2);
                const size_t slot = whole ? at + key : r.slot(u0 + key), byte = slot * 64 + 16 * part;
                k[j] = *reinterpret_cast<const uint4*>(a.c.k + byte);
                v[j] = *reinterpret_cast<const uint4*>(a.c.v + byte);
                kn[j] = a.c.ks[slot];
            }
            if (i < WD_KEYS) {
                const size_t slot = whole ? at + i : r.slot(u0 + i);
                ks = a.c.ks[slot];
                vs = a.c.vs[slot];
            }
        };
        auto store = [&](uint8_t* stage, const uint4 (&x)[2]) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int key = 32 * j + (i >> 2);
                const uint32_t c[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                uint32_t h[8];
#pragma unroll
                for (int n = 0; n < 4; n++) to_half<KIND>(c[n], h[2 * n], h[2 * n + 1]);
#pragma unroll
                for (int n = 0; n < 2; n++)
                    *reinterpret_cast<uint4*>(stage + key * 128 + (((2 * part + n) ^ (key & 7)) << 4)) =
                        make_uint4(h[4 * n], h[4 * n + 1], h[4 * n + 2], h[4 * n + 3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        // Norms of the lanes' keys (scale not included), to 2%.
        auto norm = [&](const uint4& x) {
            const uint32_t c[4] = {x.x, x.y, x.z, x.w};
            float sq;
            if (KIND == MT_KV_INT8) {
                int n = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) n = __dp4a((int)c[j], (int)c[j], n);
                sq = (float)n;
            } else {
                __half2 n = __float2half2_rn(0.f);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t h[2];
                    to_half<KIND>(c[j], h[0], h[1]);
#pragma unroll
                    for (int m = 0; m < 2; m++) {  // / 256: 16 squares stay below fp16's range
                        const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h[m]), __float2half2_rn(0x1p-8f));
                        n = __hfma2(y, y, n);
                    }
                }
                const float2 f = __half22float2(n);
                sq = (f.x + f.y + 0x1p-10f) * 65536.f;
            }
            sq += __shfl_xor_sync(0xffffffffu, sq, 1);
            sq += __shfl_xor_sync(0xffffffffu, sq, 2);
            return 1.02f * sqrtf(sq);
        };
        load(u_first);
        // The value scales' unit, from the first tile: a power of two, divided out of all of them.
        const float mine = warp_max(fabsf(vs));
        if (lane == 0) sh.first[w] = mine;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const float per_unit = power_to(fmaxf(fmaxf(sh.first[0], sh.first[1]), fmaxf(sh.first[2], sh.first[3])), 0);
        if (i == 0) sh.unit = 1.f / per_unit;
        for (int n = 0; n < tiles; n++) {
            const int st = n & (WD_STAGES - 1);
            const uint32_t reuse = ((n / WD_STAGES) & 1) ^ 1;
            const float k_top = warp_max(fmaxf(norm(k[0]) * fabsf(kn[0]), norm(k[1]) * fabsf(kn[1])));
            if (n >= WD_STAGES && !mbar_wait(&sh.k_free[st], reuse, status, 23, abort)) break;
            store(stages + st * WD_STAGE, k);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[st]);
            if (n >= WD_STAGES && !mbar_wait(&sh.v_free[st], reuse, status, 24, abort)) break;
            store(stages + (WD_STAGES + st) * WD_STAGE, v);
            if (i < WD_KEYS) {
                sh.ks[st][i] = ks;
                sh.vs[st][i] = vs * per_unit;
            }
            if (lane == 0) sh.k_top[st][w] = k_top;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[st]);
            if (n + 1 < tiles) load(u_first + (n + 1) * WD_KEYS);
        }
    } else {
        fewer_registers<WD_ISSUE_REGS>();
        if (warp == WD_ROW_WARPS + WD_CONVERT_WARPS && elect_one()) {
        const uint64_t k_desc = tile_desc(smem_u32(stages)), v_desc = tile_desc(smem_u32(stages) + WD_STAGES * WD_STAGE);
        // Scores of a row tile: 4 steps of 16 dimensions (32 bytes of a row) for each plane of Q. The lo
        // planes go first, here and below: their sums are small, and so is what the accumulator drops.
        auto scores = [&](int tile, int n) {
            const uint32_t at = tmem + tile * T_TILE;
            const uint64_t b = k_desc + (uint64_t)((n & (WD_STAGES - 1)) * (WD_STAGE >> 4));
#pragma unroll
            for (int p = 1; p >= 0; p--)
#pragma unroll
                for (int s = 0; s < 4; s++)
                    mma_ts(at + (n & 1) * WD_KEYS, at + T_Q + 16 * s + 8 * p, b + 2 * s, IDESC_S, p == 0 || s > 0);
        };
        // Outputs: 4 steps of 16 keys (16 rows of V, 2048 bytes) for each plane of P.
        auto outputs = [&](int tile, int n) {
            const uint32_t at = tmem + tile * T_TILE;
            const uint64_t b = v_desc + (uint64_t)((n & (WD_STAGES - 1)) * (WD_STAGE >> 4));
#pragma unroll
            for (int p = 1; p >= 0; p--)
#pragma unroll
                for (int s = 0; s < 4; s++)
                    mma_ts(at + T_O, at + (n & 1) * WD_KEYS + 16 * s + 8 * p, b + 128 * s, IDESC_O, p == 0 || s > 0);
        };
        auto keys_ready = [&](int n) { return mbar_wait(&sh.k_full[n & (WD_STAGES - 1)], (n / WD_STAGES) & 1, status, 25, abort); };
        bool ok = true;
        for (int n = 0; ok && n < 2 && n < tiles; n++) {
            ok = keys_ready(n);
            for (int t = 0; ok && t < row_tiles; t++) {
                ok = n > 0 || mbar_wait(&sh.q_ready[t], 0, status, 26, abort);
                if (!ok) break;
                tmem_acquire();
                scores(t, n);
                mma_done(&sh.s_ready[t][n & 1]);
            }
            if (ok) mma_done(&sh.k_free[n]);
        }
        for (int n = 0; ok && n < tiles; n++) {
            const bool more = n + 2 < tiles;
            for (int t = 0; ok && t < row_tiles; t++) {
                ok = mbar_wait(&sh.p_ready[t], n & 1, status, 27, abort) &&
                     (t > 0 || mbar_wait(&sh.v_full[n & (WD_STAGES - 1)], (n / WD_STAGES) & 1, status, 28, abort));
                if (!ok) break;
                tmem_acquire();
                outputs(t, n);
                mma_done(&sh.o_ready[t]);
                if (t == row_tiles - 1) mma_done(&sh.v_free[n & (WD_STAGES - 1)]);
                if (!more) continue;
                ok = t > 0 || keys_ready(n + 2);
                if (!ok) break;
                scores(t, n + 2);
                mma_done(&sh.s_ready[t][n & 1]);
                if (t == row_tiles - 1) mma_done(&sh.k_free[(n + 2) & (WD_STAGES - 1)]);
            }
        }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == WD_ROW_WARPS + WD_CONVERT_WARPS) {
        tmem_acquire();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace

void launch_kv8_wide(const PassArgs& a, int chunk, unsigned int* status, cudaStream_t s) {
    static PerDeviceOnce once;
    once([] {
        cudaFuncSetAttribute(kv8_wide_kernel<MT_KV_INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WD_SMEM);
        cudaFuncSetAttribute(kv8_wide_kernel<MT_KV_E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WD_SMEM);
    });
    launch_k(a.c.kind == MT_KV_INT8 ? kv8_wide_kernel<MT_KV_INT8> : kv8_wide_kernel<MT_KV_E4M3>,
             dim3((unsigned)(a.units * a.row_blocks * a.splits)), WD_THREADS, WD_SMEM, s, a, chunk, status);
}

}  // namespace mt
