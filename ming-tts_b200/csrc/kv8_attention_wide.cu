// kv8_attention_wide.cu -- attention over an 8-bit cache for many rows (prompts, batches behind a shared
// prefix) on the tcgen05 tensor cores. The arithmetic is that of kv8_attention.cu: codes exact in fp16,
// queries and weights as two fp16 planes, fp32 sums.
//
// A block takes 256 (row, head) pairs of one kv head, as two tiles of 128, and walks its keys 64 at a
// time. Its warps:
//   0-7, 8-15 the rows of tile 0, 1 (16 a warp): they read scores from TMEM, keep each row's reference and
//             sum, write the weights (times the value rows' scales) back as two fp16 planes over the
//             scores, and add each key tile's output, read from TMEM, to registers
//   16-18     convert codes to fp16 in shared memory (four stages), K and V alike: a key a 128-byte row
//   19        issues the matrix instructions: S = Q K^T (128 x 64, both planes of Q in shared memory) and
//             O = P V (128 x 64, both planes of P in TMEM; V is the [key][dimension] tile as it is)
// Scores and outputs have two buffers each: the scores of the next key tile are there while a tile's
// weights are made, and an output is read two tiles later, so neither the row warps nor the tensor cores
// wait for the other in turn. (With one output buffer and the query planes in TMEM, a tile had to wait
// for the product of the one before: 2800 cycles a key tile even with no arithmetic on the weights.)
//
// Every key tile's O starts from zero: the accumulators drop the bits that 24 do not hold, and a chain of
// 64 keys keeps that near fp32's own rounding; it also leaves nothing in TMEM to rescale.
//
// TMEM, 256 columns a row tile: 0-63 and 64-127 scores of even and odd key tiles (fp32), overwritten 16
// columns at a time by 8 columns of hi and 8 of lo planes of the same 16 keys' weights; 128-191 and
// 192-255 their outputs.
//
// A row warp has 16 of the 32 lanes that its place in the block lets it read, in the layout of 16 rows x 8
// columns to 4 registers: lane (g, t) = (lane / 4, lane % 4) has columns 2t, 2t+1 of every 8, of rows g
// and g + 8 (its slots 0 and 1). Four such warps a scheduler hide one another's latencies: with 8 warps of
// 32 rows a key tile took 3400 cycles, of which 2200 were these warps' own.
//
// Bounded by the row warps: 21 instructions a score, two thirds of the SM's issue slots, the rest their waits for TMEM
// and for one another; 16 bytes a thread of the 96 registers spill, beside the loops. 2.2 us for 64 keys of 256 rows in
// the steady state, 14 us more for a block's start and end. 4096 rows over themselves, 14 heads on 2, e4m3: 130 us,
// 464 TFLOP/s of matrix work in two planes; the warp kernel took 304. The same with int8, 5 instructions for 4 codes
// instead of 2, takes 157 us.
#include <math.h>

#include "kv8.cuh"

namespace mt {

namespace {

constexpr int WD_ROW_WARPS = 16, WD_CONVERT_WARPS = 3;
constexpr int WD_THREADS = 32 * (WD_ROW_WARPS + WD_CONVERT_WARPS + 1);
// Registers of a thread, by warpgroup: the block starts with 640 x 96 = 61,440 of them, and
// 512 x 104 + 128 x 64 is as many.
constexpr int WD_ROW_REGS = 104, WD_OTHER_REGS = 64;
constexpr int WD_KEYS = KV8_WIDE_KEYS;
constexpr int WD_STAGE = WD_KEYS * 128;  // bytes of a K or V tile in fp16
constexpr int WD_STAGES = 4;
constexpr int WD_PLANE = 128 * 128;      // bytes of a plane of a row tile's queries
constexpr size_t WD_SMEM = 2 * WD_STAGES * WD_STAGE + 4 * WD_PLANE + 1024;
constexpr uint32_t T_O = 128, T_TILE = 256;
// 16 lanes x 16 columns of TMEM to and from 8 registers: fp32 (register 4 n + 2 slot + i is column 8 n + 2 t
// + i of row g + 8 slot) or fp16 pairs (register 2 n + slot is column 4 n + t). A load's registers are
// operands of the wait for it, so that nothing uses them before.
#define TM_OUT8(r) "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
__device__ __forceinline__ void tmem_ld_tile(uint32_t at, float (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : TM_OUT8(r) : "r"(at));
}
__device__ __forceinline__ void tmem_ld_planes(uint32_t at, float (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x128b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : TM_OUT8(r) : "r"(at));
}
__device__ __forceinline__ void tmem_ld_wait(float (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st_planes(uint32_t at, const uint32_t (&u)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(u[0]), "r"(u[1]),
                 "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// TMEM stores of this thread done and ordered before what another thread does after a barrier.
__device__ __forceinline__ void tmem_publish() {
    tmem_st_wait();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_acquire() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D[tmem] (+)= A B, A in TMEM or in shared memory, B in shared memory; fp16 operands, fp32 accumulator,
// M = 128.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
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
    alignas(16) float ks[WD_STAGES][WD_KEYS], vs[2][WD_STAGES][WD_KEYS];  // scales of the stages' keys; values': times 2^unit, and as they are
    float first[WD_CONVERT_WARPS];
    float unit;                                                        // brings the first value scales near 1
    uint64_t k_full[WD_STAGES], k_free[WD_STAGES], v_full[WD_STAGES], v_free[WD_STAGES];
    uint64_t q_ready[2], s_ready[2][2], p_ready[2][2], o_ready[2][2];     // by row tile (and key tile parity)
    uint64_t idle;                                                        // all matrix instructions are done
    uint32_t tmem;
    int abort, never;  // never stays 0: for the wait that goes on after an abort
};

// Units of rows (see kv8_move). The factor 2^unit is in the value scales already, for all rows of a block; a row's lift
// does the rest up to 2^16 either way, at the price of the exponents' rounding to 2^-20, and the fast path knows no
// other. Rows whose first values are further from the first of the block, or whose scores have no fraction in fp32
// (see kv8_score), go the slow way, with an extra of their own.
constexpr float WD_LIFT = 16.f, WD_LARGEST = 0x1p127f;
__device__ __forceinline__ float row_lift(float total, float unit) { return fminf(WD_LIFT, fmaxf(-WD_LIFT, total - unit)); }
__device__ __forceinline__ float row_extra(float total, float unit) {
    if (total == KV8_UNSET) return 1.f;
    return kv8_power(total > 0.5f * KV8_FAR ? total - KV8_FAR : total - row_lift(total, unit));
}
__device__ __forceinline__ bool row_usual(float off, float total, float unit) { return fabsf(total - unit) <= WD_LIFT && fabsf(off) < 0x1p24f; }
// Not that far, but without products that count (yet).
__device__ __forceinline__ bool row_plain(float off, float total, float unit) {
    return (total == KV8_UNSET || fabsf(total - unit) <= WD_LIFT) && (off == KV8_REF_NONE || fabsf(off) < 0x1p24f);
}

// The state of a lane's two rows; off and total: see kv8_move. A sum is the lane's own part of the row.
struct RowState {
    float off[2], total[2], rs[2];  // rs: scores in powers of two are TMEM value x key scale x rs
    int lo[2], hi[2];              // keys that the row sees
    float sum[2];
    float o[4][8];  // 16 columns each, as tmem_ld_tile
    bool usual;     // all rows of the warp are: see row_usual

    __device__ __forceinline__ void scale(int slot, const Kv8Move& move) {
        const float f = move.outputs;
        sum[slot] *= move.sums;
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                o[c][4 * n + 2 * slot] *= f;
                o[c][4 * n + 2 * slot + 1] *= f;
            }
    }
};

// The keys of a tile: the lane's first scales in shared memory (its columns are 8 n + 0, 1 from there),
// and their index.
struct TileKeys {
    const float *ks, *vs;
    int u;
    const float* at_unit;
    __device__ __forceinline__ float unit() const { return *reinterpret_cast<const volatile float*>(at_unit); }
    __device__ __forceinline__ const float* raw() const { return vs + WD_STAGES * WD_KEYS; }  // the values' as they are
};

// The planes of `chunks` times 16 keys, scaled by the rows' factors.
__device__ __forceinline__ void row_rescale(uint32_t tm, int chunks, float f0, float f1) {
    tmem_st_wait();
#pragma unroll 1
    for (int c = 0; c < chunks; c++) {
        float x[8];
        uint32_t planes[8];
        tmem_ld_planes(tm + 16 * c, x);
        tmem_ld_wait(x);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = j & 1 ? f1 : f0;
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&x[j]));
            const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&x[4 + j]));
            split_half2((hi.x + lo.x) * f, (hi.y + lo.y) * f, planes[j], planes[4 + j]);
        }
        tmem_st_planes(tm + 16 * c, planes);
        tmem_st_wait();
    }
}

// Weights of 16 keys (s: scores, k and v: the keys' scales): 2^(score - off), their sums, and times the
// value scales as planes. MASK: rows see some of the keys; OWN: units are the rows' own. Returns the largest product.
template <bool MASK, bool OWN>
__device__ __forceinline__ float row_products(const TileKeys& t, const RowState& row, int c, const float (&s)[8], uint32_t (&planes)[8],
                                              float (&add)[2]) {
    const float2 k[2] = {*reinterpret_cast<const float2*>(t.ks + 16 * c), *reinterpret_cast<const float2*>(t.ks + 16 * c + 8)};
    const float* const vs = (OWN ? t.raw() : t.vs) + 16 * c;
    const float2 v[2] = {*reinterpret_cast<const float2*>(vs), *reinterpret_cast<const float2*>(vs + 8)};
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float sum[2];
        const float extra = OWN ? row_extra(row.total[i], t.unit()) : 1.f;
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int u = t.u + 16 * c + 8 * n;
            const bool on0 = !MASK || (u >= row.lo[i] && u <= row.hi[i]), on1 = !MASK || (u + 1 >= row.lo[i] && u + 1 <= row.hi[i]);
            // key scale and rs first: see kv8_attention.cu
            const float k0 = k[n].x * row.rs[i], k1 = k[n].y * row.rs[i], s0 = s[4 * n + 2 * i], s1 = s[4 * n + 2 * i + 1];
            float p0 = ex2(OWN ? kv8_score(s0, k0) - row.off[i] : fmaf(s0, k0, -row.off[i]));
            float p1 = ex2(OWN ? kv8_score(s1, k1) - row.off[i] : fmaf(s1, k1, -row.off[i]));
            if (MASK) {
                p0 = on0 ? p0 : 0.f;
                p1 = on1 ? p1 : 0.f;
            }
            sum[n] = p0 + p1;
            p0 *= v[n].x;
            p1 *= v[n].y;
            if (OWN) {
                p0 *= extra;
                p1 *= extra;
            }
            if (MASK) {  // a scale of a key that this row does not see may be NaN
                p0 = on0 ? p0 : 0.f;
                p1 = on1 ? p1 : 0.f;
            }
            top = fmaxf(top, fmaxf(fabsf(p0), fabsf(p1)));
            split_half2(p0, p1, planes[2 * n + i], planes[4 + 2 * n + i]);
        }
        add[i] = sum[0] + sum[1];
    }
    return top;
}

// A tile whose keys all rows see and whose products stay in range: nothing here changes a row's units,
// which is what keeps the loop at 9.4 instructions a weight (with that code in it, 12). Returns the first
// 16 keys whose products do not stay in range, or 4.
__device__ __forceinline__ int row_weights(uint32_t tm, const TileKeys& t, RowState& row) {
    int c;
#pragma unroll 1
    for (c = 0; c < 4; c++) {
        float s[8], add[2];
        uint32_t planes[8];
        tmem_ld_tile(tm + 16 * c, s);
        tmem_ld_wait(s);
        const float top = row_products<false, false>(t, row, c, s, planes, add);
        if (__any_sync(0xffffffffu, !(top <= KV8_PRODUCT_MAX && add[0] <= KV8_WEIGHT_MAX && add[1] <= KV8_WEIGHT_MAX))) break;
        row.sum[0] += add[0];
        row.sum[1] += add[1];
        tmem_st_planes(tm + 16 * c, planes);
    }
    return c;
}

// The rest of a tile from `c` on, whatever its rows see and their units are: sets those of rows that have none, and
// moves them where products leave the range. `settle` adds the outputs that are still in TMEM, which are in the
// units before.
template <typename F>
__device__ __forceinline__ void row_weights_slowly(uint32_t tm, const TileKeys& t, RowState& row, int c, F&& settle) {
#pragma unroll 1
    for (; c < 4; c++) {
        float s[8], add[2];
        uint32_t planes[8];
        tmem_ld_tile(tm + 16 * c, s);
        tmem_ld_wait(s);
#pragma unroll 1
        for (bool move = !row.usual && __any_sync(0xffffffffu, row.total[0] == KV8_UNSET || row.total[1] == KV8_UNSET);; move = true) {
            if (move) {
                settle(1);
                float f[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float z[4], v[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = 16 * c + 8 * (j >> 1) + (j & 1);
                        const bool on = t.u + key >= row.lo[i] && t.u + key <= row.hi[i];
                        z[j] = on ? kv8_score(s[4 * (j >> 1) + 2 * i + (j & 1)], t.ks[key] * row.rs[i]) : -INFINITY;
                        v[j] = on ? fabsf(t.raw()[key]) : 0.f;
                    }
                    const Kv8Move by = kv8_move(z, v, row.off[i], row.total[i], [&](float total) { return row_lift(total, t.unit()); });
                    if (by.sums != 1.f || by.outputs != 1.f) row.scale(i, by);
                    f[i] = by.outputs;
                }
                row.usual = __all_sync(0xffffffffu, row_usual(row.off[0], row.total[0], t.unit()) && row_usual(row.off[1], row.total[1], t.unit()));
                row_rescale(tm, c, f[0], f[1]);
            }
            float top;
            if (row.usual || __all_sync(0xffffffffu, row_plain(row.off[0], row.total[0], t.unit()) && row_plain(row.off[1], row.total[1], t.unit())))
                top = row_products<true, false>(t, row, c, s, planes, add);
            else
                top = row_products<true, true>(t, row, c, s, planes, add);
            if (move || !__any_sync(0xffffffffu, !(top <= KV8_PRODUCT_MAX && add[0] <= KV8_WEIGHT_MAX && add[1] <= KV8_WEIGHT_MAX))) break;
        }
        row.sum[0] += add[0];
        row.sum[1] += add[1];
        tmem_st_planes(tm + 16 * c, planes);
    }
}

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int KIND>
__device__ __forceinline__ void wide_block(const PassArgs& a, int chunk, unsigned int* status) {
    extern __shared__ uint8_t dynamic[];
    __shared__ Shared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Blocks with the most keys (the last rows) first.
    const int split = blockIdx.x % a.splits;
    const int unit = (blockIdx.x / a.splits) % a.units;
    const int row_block = a.row_blocks - 1 - blockIdx.x / (a.splits * a.units);
    UnitRows rows(a, unit);
    pass_begin(a.beside);
    rows.locate();
    const int e0 = row_block * KV8_WIDE_ROWS, left = rows.size() - e0;
    if (left <= 0) return;
    rows.tile(e0, KV8_WIDE_ROWS);
    const KeyRange& r = rows.keys;
    const int u_first = (r.lo & ~15) + split * chunk * WD_KEYS;
    const int tiles = min(chunk, (r.hi - u_first) / WD_KEYS + 1);  // of this part
    if (u_first > r.hi) {
        if (warp < WD_ROW_WARPS) {
            int lo, hi;
            const int target = threadIdx.x < KV8_WIDE_ROWS ? rows.pair(e0 + threadIdx.x, lo, hi) : -1;
            if (target >= 0)
                reinterpret_cast<float2*>(a.part_ml)[a.part0 + (size_t)target * a.splits + split] = make_float2(KV8_REF_NONE, 0.f);
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
            mbar_init(&sh.q_ready[i], WD_ROW_WARPS / 2);
            mbar_init(&sh.s_ready[i][0], 1);
            mbar_init(&sh.s_ready[i][1], 1);
            mbar_init(&sh.p_ready[i][0], WD_ROW_WARPS / 2);
            mbar_init(&sh.p_ready[i][1], WD_ROW_WARPS / 2);
            mbar_init(&sh.o_ready[i][0], 1);
            mbar_init(&sh.o_ready[i][1], 1);
        }
        mbar_init(&sh.idle, 1);
        sh.abort = sh.never = 0;
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

    if (warp >= WD_ROW_WARPS) fewer_registers<WD_OTHER_REGS>();
    if (warp < WD_ROW_WARPS) {
        more_registers<WD_ROW_REGS>();
        const int tile = warp >> 3;
        if (tile < row_tiles) {
            const int first_row = 32 * (warp & 3) + 16 * ((warp >> 2) & 1);  // of the tile's 128: a lane of TMEM each
            const uint32_t tm = tmem + tile * T_TILE + ((uint32_t)first_row << 16);
            const int col = 2 * (lane & 3);
            int target[2];
            RowState row;
            {
                // Queries: a lane has dimensions 8 n + 2 t, + 1 of its two rows.
                int lo, hi;
                const int mine = rows.pair(e0 + 128 * tile + first_row + (lane & 15), lo, hi), at = mine / a.hq;
                long long from = (long long)at * a.ldq + (long long)(mine - at * a.hq) * 64;
                if (mine < 0) from = -1;
                const float* src[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int owner = 8 * i + (lane >> 2);
                    target[i] = __shfl_sync(0xffffffffu, mine, owner);
                    row.lo[i] = __shfl_sync(0xffffffffu, lo, owner);
                    row.hi[i] = __shfl_sync(0xffffffffu, hi, owner);
                    src[i] = a.q + __shfl_sync(0xffffffffu, from, owner) + col;
                }
                float2 x[2][8];
                if (a.qvec) {  // all of them issued before the first is used
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        x[j >> 3][j & 7] = target[j >> 3] < 0 ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(src[j >> 3] + 8 * (j & 7));
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        x[j >> 3][j & 7] = target[j >> 3] < 0 ? make_float2(0.f, 0.f) : make_float2(src[j >> 3][8 * (j & 7)], src[j >> 3][8 * (j & 7) + 1]);
                }
                float top[2] = {0.f, 0.f}, up[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
#pragma unroll
                    for (int n = 0; n < 8; n++) top[i] = fmaxf(top[i], fmaxf(fabsf(x[i][n].x), fabsf(x[i][n].y)));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
                    up[i] = power_to(top[i], 13);
                    const int at = first_row + 8 * i + (lane >> 2);
                    uint8_t* to = stages + 2 * WD_STAGES * WD_STAGE + 2 * tile * WD_PLANE + at * 128 + 2 * col;
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        const float x0 = x[i][n].x * up[i], x1 = x[i][n].y * up[i];
                        uint8_t* const here = to + ((n ^ (at & 7)) << 4);
                        split_half2(x0, x1, *reinterpret_cast<uint32_t*>(here), *reinterpret_cast<uint32_t*>(here + WD_PLANE));
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    // up is a power of two within 2^+-126: so is its reciprocal
                    row.rs[i] = 0.125f * 1.4426950408889634f * __uint_as_float(0x7F000000u - __float_as_uint(up[i]));
                    row.off[i] = KV8_REF_NONE;
                    row.total[i] = KV8_UNSET;
                    row.sum[i] = 0.f;
                }
                row.usual = false;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_ready[tile]);

#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) row.o[c][j] = 0.f;
            bool ok = true;
            int n = 0, added = 0;  // key tiles begun, and those whose output is in row.o
            auto settle = [&](int back) {
#pragma unroll 1
                for (; added <= n - back && ok; added++) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_ready[tile][added & 1], (added >> 1) & 1, status, 22, abort));
                    if (!ok) return;
                    tmem_acquire();
                    const uint32_t from = tm + T_O + (added & 1) * 64;
                    float y[2][8];
                    tmem_ld_tile(from, y[0]);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        tmem_ld_wait(y[c & 1]);
                        if (c < 3) tmem_ld_tile(from + 16 * c + 16, y[(c + 1) & 1]);
#pragma unroll
                        for (int j = 0; j < 8; j++) row.o[c][j] += y[c & 1][j];
                    }
                }
            };
            for (; ok && n < tiles; n++) {
                const int st = n & (WD_STAGES - 1), u0 = u_first + n * WD_KEYS;
                ok = mbar_wait(&sh.v_full[st], (n / WD_STAGES) & 1, status, 21, abort) &&  // the scales come with the values
                     mbar_wait(&sh.s_ready[tile][n & 1], (n >> 1) & 1, status, 20, abort);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tmem_acquire();
                const TileKeys keys{sh.ks[st] + col, sh.vs[0][st] + col, u0 + col, &sh.unit};
                const uint32_t tp = tm + (n & 1) * WD_KEYS;
                settle(2);
                int c = 0;
                if (row.usual && u0 >= r.in_lo && u0 + WD_KEYS - 1 <= r.in_hi) c = row_weights(tp, keys, row);
                if (c < 4) row_weights_slowly(tp, keys, row, c, settle);
                tmem_publish();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready[tile][n & 1]);  // by parity: a warp can be a tile ahead of another
            }
            if (ok) settle(1);
            if (ok) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float s0 = row.sum[i];
                    s0 += __shfl_xor_sync(0xffffffffu, s0, 1);
                    s0 += __shfl_xor_sync(0xffffffffu, s0, 2);
                    if (target[i] < 0) continue;
                    const OverSum out(row_extra(row.total[i], sh.unit), s0);
                    float* dst;
                    bool vec = true;
                    if (!a.parted) {
                        const int at = target[i] / a.hq;
                        dst = a.out + (size_t)at * a.ldo + (size_t)(target[i] - at * a.hq) * 64;
                        vec = a.ovec;
                    } else {
                        const size_t at = (size_t)target[i] * a.splits + a.part0 + split;
                        if (col == 0) reinterpret_cast<float2*>(a.part_ml)[at] = kv8_total(row.off[i], s0);
                        dst = a.part_o + at * 64;
                    }
                    dst += col;
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float* o = row.o[c] + 4 * j + 2 * i;
                            if (vec) {
                                *reinterpret_cast<float2*>(dst + 16 * c + 8 * j) = make_float2(out(o[0]), out(o[1]));
                            } else {
                                dst[16 * c + 8 * j] = out(o[0]);
                                dst[16 * c + 8 * j + 1] = out(o[1]);
                            }
                        }
                }
            }
        }
    } else if (warp < WD_ROW_WARPS + WD_CONVERT_WARPS) {
        // Four lanes a key, 16 codes each: 8 keys a warp at a time, the three warps in turn. The stages let
        // them run ahead of the tensor cores, which hides the loads' latency.
        const int w = warp - WD_ROW_WARPS, part = lane & 3;
        constexpr int TURNS = (WD_KEYS / 8 + WD_CONVERT_WARPS - 1) / WD_CONVERT_WARPS;
        uint4 k[TURNS], v[TURNS];
        float ks[TURNS], vs[TURNS];
        auto key_of = [&](int j) { return 8 * (w + WD_CONVERT_WARPS * j) + (lane >> 2); };
        const uint8_t *k0 = a.c.k + r.row * 64 + 16 * part, *v0 = a.c.v + r.row * 64 + 16 * part;
        const float *ks0 = a.c.ks + r.row, *vs0 = a.c.vs + r.row;
        auto load = [&](int u0) {
            const bool whole = r.whole(u0, WD_KEYS);
            const int first = u0 >= r.capacity ? u0 - r.capacity : u0;
#pragma unroll
            for (int j = 0; j < TURNS; j++) {
                // Keys outside the range stand in as the nearest inside it: see kv8_attention.cu.
                const int key = min(key_of(j), WD_KEYS - 1);
                int slot = first + key;
                if (!whole) {
                    slot = min(max(u0 + key, r.lo), r.hi);
                    slot = slot >= r.capacity ? slot - r.capacity : slot;
                }
                k[j] = *reinterpret_cast<const uint4*>(k0 + (size_t)slot * 64);
                v[j] = *reinterpret_cast<const uint4*>(v0 + (size_t)slot * 64);
                ks[j] = ks0[slot];
                vs[j] = vs0[slot];
            }
        };
        auto store = [&](uint8_t* stage, const uint4 (&x)[TURNS]) {
#pragma unroll
            for (int j = 0; j < TURNS; j++) {
                const int key = key_of(j);
                if (key >= WD_KEYS) break;
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
        load(u_first);
        // The value scales' unit, from the first tile (all zero: none).
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < TURNS; j++) most = fmaxf(most, fabsf(vs[j]));
        most = warp_max(most);
        if (lane == 0) sh.first[w] = most;
        asm volatile("bar.sync 1, 96;" ::: "memory");
        most = fmaxf(sh.first[0], fmaxf(sh.first[1], sh.first[2]));
        const float per_unit = most > 0.f ? power_to(most, 0) : 1.f;
        if (w == 0 && lane == 0) sh.unit = (float)((int)(__float_as_uint(per_unit) >> 23) - 127);
        for (int n = 0; n < tiles; n++) {
            if (n > 0) load(u_first + n * WD_KEYS);
            const int st = n & (WD_STAGES - 1);
            const uint32_t reuse = ((n / WD_STAGES) & 1) ^ 1;
            // A wait that gives up ends the loop for the whole warp: its lanes meet again below.
            if (n >= WD_STAGES && !__all_sync(0xffffffffu, mbar_wait(&sh.k_free[st], reuse, status, 23, abort))) break;
            store(stages + st * WD_STAGE, k);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[st]);
            if (n >= WD_STAGES && !__all_sync(0xffffffffu, mbar_wait(&sh.v_free[st], reuse, status, 24, abort))) break;
            store(stages + (WD_STAGES + st) * WD_STAGE, v);
            if (part == 0) {
#pragma unroll
                for (int j = 0; j < TURNS; j++) {
                    const int key = key_of(j);
                    if (key >= WD_KEYS) break;
                    sh.ks[st][key] = ks[j];
                    // Not infinite, so that a weight of 0 does not make it NaN. A usual row's largest weight is 2^-16 or
                    // more, and one of 2^-112 times this is a product that goes the slow way.
                    const float near1 = vs[j] * per_unit;
                    sh.vs[0][st][key] = near1 > WD_LARGEST ? WD_LARGEST : near1;
                    sh.vs[1][st][key] = vs[j];
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[st]);
        }
    } else {
        if (warp == WD_ROW_WARPS + WD_CONVERT_WARPS && elect_one()) {
        const uint64_t k_desc = tile_desc(smem_u32(stages)), v_desc = tile_desc(smem_u32(stages) + WD_STAGES * WD_STAGE);
        const uint64_t q_desc = tile_desc(smem_u32(stages) + 2 * WD_STAGES * WD_STAGE);
        // Scores of a row tile: 4 steps of 16 dimensions (32 bytes of a row) for each plane of Q. The lo
        // planes go first, here and below: their sums are small, and so is what the accumulator drops.
        auto scores = [&](int tile, int n) {
            const uint32_t at = tmem + tile * T_TILE;
            const uint64_t b = k_desc + (uint64_t)((n & (WD_STAGES - 1)) * (WD_STAGE >> 4));
            const uint64_t q = q_desc + (uint64_t)(tile * (2 * WD_PLANE >> 4));
#pragma unroll
            for (int p = 1; p >= 0; p--)
#pragma unroll
                for (int s = 0; s < 4; s++)
                    mma_ss(at + (n & 1) * WD_KEYS, q + p * (WD_PLANE >> 4) + 2 * s, b + 2 * s, IDESC_S, p == 0 || s > 0);
        };
        // Outputs: 4 steps of 16 keys (16 rows of V, 2048 bytes) for each plane of P.
        auto outputs = [&](int tile, int n) {
            const uint32_t at = tmem + tile * T_TILE;
            const uint64_t b = v_desc + (uint64_t)((n & (WD_STAGES - 1)) * (WD_STAGE >> 4));
#pragma unroll
            for (int p = 1; p >= 0; p--)
#pragma unroll
                for (int s = 0; s < 4; s++)
                    mma_ts(at + T_O + (n & 1) * 64, at + (n & 1) * WD_KEYS + 16 * s + 8 * p, b + 128 * s, IDESC_O, p == 0 || s > 0);
        };
        auto keys_ready = [&](int n) { return mbar_wait(&sh.k_full[n & (WD_STAGES - 1)], (n / WD_STAGES) & 1, status, 25, abort); };
        bool ok = true;
        for (int t = 0; ok && t < row_tiles; t++) ok = mbar_wait(&sh.q_ready[t], 0, status, 26, abort);
        for (int n = -1; ok && n < tiles; n++) {
            // The next tile's scores, into the buffer of the last one's weights: its product has read them.
            if (n + 1 < tiles) {
                ok = keys_ready(n + 1);
                for (int t = 0; ok && t < row_tiles; t++) {
                    ok = n < 1 || mbar_wait(&sh.o_ready[t][(n - 1) & 1], ((n - 1) >> 1) & 1, status, 30, abort);
                    if (!ok) break;
                    tmem_acquire();
                    scores(t, n + 1);
                    mma_done(&sh.s_ready[t][(n + 1) & 1]);
                }
                if (ok) mma_done(&sh.k_free[(n + 1) & (WD_STAGES - 1)]);
            }
            if (n < 0 || !ok) continue;
            ok = mbar_wait(&sh.v_full[n & (WD_STAGES - 1)], (n / WD_STAGES) & 1, status, 28, abort);
            for (int t = 0; ok && t < row_tiles; t++) {
                ok = mbar_wait(&sh.p_ready[t][n & 1], (n >> 1) & 1, status, 27, abort);
                if (!ok) break;
                tmem_acquire();
                outputs(t, n);
                mma_done(&sh.o_ready[t][n & 1]);
            }
            if (ok) mma_done(&sh.v_free[n & (WD_STAGES - 1)]);
        }
        // Also after a wait that gave up: shared memory and TMEM stay until nothing uses them.
        mma_done(&sh.idle);
        mbar_wait(&sh.idle, 0, status, 29, &sh.never);
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

template <int KIND>
__global__ void __launch_bounds__(WD_THREADS, 1) kv8_wide_kernel(const PassArgs a, int chunk, unsigned int* status) {
    wide_block<KIND>(a, chunk, status);
    if (a.beside) pdl_wait();
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
