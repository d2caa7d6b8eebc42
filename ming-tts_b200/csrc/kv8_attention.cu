// kv8_attention.cu -- attention over 8-bit key/value caches, alone (mt_attention_kv8) and behind a
// prefix that all requests share (mt_attention_prefix_kv8).
//
// out = sum_j w_j v_j / sum_j w_j with w_j = exp(q.k_j / 8 - m), one pass with a running reference m.
// The reference's attention_cache (Shaders.swift:500-591) reads fp32 caches of one request.
//
// Arithmetic. A code (an integer up to 128, or an e4m3 value) is exact in fp16. A query value and a
// weight (times its value row's scale) are carried as two fp16 planes, x = hi + lo with
// |x - hi - lo| <= 2^-22 |x|, so two 16-bit matrix products with fp32 sums give both contractions at
// fp32 accuracy: q.k_j = scale_j (hi.c_j + lo.c_j), and the same for the values. Queries are scaled by
// a power of two per row, products of weights and value scales by one per row that follows the largest, so
// that the planes use fp16's range whatever the units (kv8_move).
//
// A warp owns a tile of 8 query rows (rows x grouped heads, flattened) and walks its keys 16 at a time, copied
// ahead into a ring in shared memory. The rows' hi planes are rows 0-7 and their lo planes rows 8-15 of the
// 16-row operand of m16n8k16, for the queries and again for the weights. Which key or dimension a fragment's
// row or column stands for is free as long as both operands agree, so a lane takes 16 consecutive bytes of
// one key row for the scores, 8 consecutive bytes of four key rows for the values, and the conversion to
// fp16 pairs the bytes of two keys. Warps meet only when the partial results of a block are merged.
//   Lane (g, t) = (lane / 4, lane % 4), in a tile of keys 0..15:
//     scores, column g of half j is key 4 (g / 2) + 2 j + g % 2, so lane t's scores are keys 4t .. 4t+3
//     values, contraction index 2t, 2t+1, 2t+8, 2t+9 is key 4t .. 4t+3; column g of block i is dimension
//     8 g + i, so lane t's outputs are dimensions 16 t .. 16 t + 15.
// Bounded by latency: a warp is one chain of dependent steps a key tile (codes, conversion, scores, exponentials,
// planes, products), and registers leave 4 warps a scheduler. 64 requests of 8000 keys take 43 us, half of the copy
// bandwidth: 336 instructions a tile of 16 keys (16 matrix instructions, some 90 to convert codes) use 56% of the issue
// slots, and a warp waits 1.7 cycles an instruction for the fixed latency of the one before, 0.6 each for the matrix
// unit and shared memory. Tiles of 16 and 32 rows (the planes as operands of their own, each code converted once
// for all of them) were no faster at any size: 974 instructions a tile of 32, but registers for 8 warps an
// SM, which used 40% of the slots, and 16 rows over 300 keys took 9.1 and 13.6 us instead of 6.3. Many rows
// against many keys go to kv8_attention_wide.cu.
#include <math.h>

#include <type_traits>

#include "kv8.cuh"

namespace mt {

namespace {

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A warp's ring of key tiles in shared memory, filled by asynchronous copies RING - 1 tiles ahead: codes of
// 16 keys (64 bytes a key) and their scales. 16 warps an SM have some 100 KB in flight, where one tile
// ahead in registers had 33 and was bound by DRAM's latency (8 long requests 28 us).
constexpr int RING = 4;
constexpr int TILE_BYTES = 2 * 16 * 64 + 2 * 16 * 4;

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool l1) {
    if (l1) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// Keys outside the range stand in as the nearest inside it: the slot of a key that no row sees may hold
// codes that are NaN, which a weight of zero would not silence. Value rows are placed so that the reads
// below (4 rows 256 bytes apart, 8 bytes each of 4 places) touch every bank once: odd groups of four rows
// have their rows swapped in pairs, the last eight rows their halves.
struct KeyCopy {
    const uint8_t *k, *v;  // this lane's first: row lane / 4, 16 bytes at lane % 4
    const float* scale;    // key lane % 16, of the keys (lanes 0-15) or values
    uint32_t to_k, to_v, to_scale;
    bool l1;

    __device__ __forceinline__ KeyCopy(const Kv8View& c, const KeyRange& r, uint32_t ring, int lane, bool l1_) : l1(l1_) {
        const int part = lane & 3, row = lane >> 2;
        k = c.k + (r.row + row) * 64 + 16 * part;
        v = c.v + (r.row + row) * 64 + 16 * part;
        scale = (lane < 16 ? c.ks : c.vs) + r.row + (lane & 15);
        to_k = ring + row * 64 + 16 * part;
        to_v = ring + 1024 + (row ^ ((row >> 2) & 1)) * 64 + 16 * part;
        to_scale = ring + 2048 + 4 * lane;
    }
    __device__ __forceinline__ void tile(const KeyRange& r, int u0, int stage, int lane) const {
        const uint32_t at = stage * TILE_BYTES;
        int slot[2], key;  // less the lane's own row
        if (r.whole(u0, 16)) {
            slot[0] = u0 >= r.capacity ? u0 - r.capacity : u0;
            slot[1] = slot[0] + 8;
            key = slot[0];
        } else {
            auto nearest = [&](int n) {
                const int u = min(max(u0 + n, r.lo), r.hi);
                return (u >= r.capacity ? u - r.capacity : u) - n;
            };
            slot[0] = nearest(lane >> 2);
            slot[1] = nearest((lane >> 2) + 8) + 8;
            key = nearest(lane & 15);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            copy16(to_k + at + 512 * j, k + (long long)slot[j] * 64, l1);
            copy16((to_v ^ (32 * j)) + at + 512 * j, v + (long long)slot[j] * 64, l1);
        }
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to_scale + at), "l"(scale + key) : "memory");
    }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int ROWS = 8, WARPS = 8;  // rows of a warp, warps of a block (two blocks an SM)
constexpr int SUM_BYTES = WARPS * ROWS * (64 + 4 + 1) * 4;  // sums, references and factors, owners
constexpr int SMEM = SUM_BYTES + WARPS * RING * TILE_BYTES;
constexpr int FOLD = 8;               // key tiles summed in the matrix unit's accumulators at a time

// The slots of a kv head (and row block) are shared out so that the longest walk is the shortest: requests
// get ceil(rounds / q) each, with the smallest q that the slots allow, a round being a key tile for each of
// the block's warps. Every block computes the same from all positions. With an equal number of slots each,
// 8 requests of 4000 to 32768 keys took 23.1 us, nearly as long as 8 of 32000; so they took 19.4.
constexpr int SHARE_LANES = 5;  // requests per lane at most
struct Share {
    int request, first, parts;  // parts 0: no request's slot
};
__device__ __forceinline__ Share share_of(const PassArgs& a, int slot, int lane) {
    float rounds[SHARE_LANES];  // less a half: ceil(n / q) = floor((n - 1/2) / q) + 1, exact in fp32 up to 2^21
    int total = 0, most = 0;
#pragma unroll
    for (int j = 0; j < SHARE_LANES; j++) {
        rounds[j] = -1.f;
        const int request = 32 * j + lane;
        if (32 * j >= a.requests) break;
        if (request < a.requests) {
            const Kv8Span s = kv8_span(a.rows, request);
            int keys = min(s.pos + s.count - a.rows.base, a.c.capacity);
            if (a.window > 0) keys = min(keys, a.window + s.count - 1);
            const int n = s.count > 0 ? (keys + 15 + 16 * a.key_warps) / (16 * a.key_warps) : 0;
            rounds[j] = (float)n - 0.5f;
            total += n;
            most = max(most, n);
        }
    }
    total = __reduce_add_sync(0xffffffffu, total);
    most = __reduce_max_sync(0xffffffffu, most);
    auto parts = [&](int j, float one_over) { return rounds[j] < 0.f ? 0 : (int)(rounds[j] * one_over) + 1; };
    // A part a request is allowed, and so is what leaves each request one slot to round up into.
    int lo = max(2, (total + a.slots - 1) / a.slots);
    int hi = max(lo, min(most, (total + a.slots - a.requests - 1) / (a.slots - a.requests)));
#pragma unroll 1
    for (int i = 0; i < 4 && lo < hi; i++) {
        const int q = (lo + hi) >> 1;
        const float one_over = __frcp_rn((float)q);
        int n = 0;
#pragma unroll
        for (int j = 0; j < SHARE_LANES; j++) {
            if (32 * j >= a.requests) break;
            n += parts(j, one_over);
        }
        if (__reduce_add_sync(0xffffffffu, n) <= a.slots) hi = q;
        else lo = q + 1;
    }
    const float one_over = __frcp_rn((float)hi);
    Share mine{0, 0, 0};
    int before = 0;
#pragma unroll
    for (int j = 0; j < SHARE_LANES; j++) {
        if (32 * j >= a.requests) break;
        const int n = parts(j, one_over);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const uint32_t here = __ballot_sync(0xffffffffu, before + upto > slot && before + upto - n <= slot && n > 0);
        if (here) {
            const int from = __ffs(here) - 1;
            mine.request = 32 * j + from;
            mine.parts = __shfl_sync(0xffffffffu, n, from);
            mine.first = before + __shfl_sync(0xffffffffu, upto, from) - mine.parts;
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return mine;
}

template <int KIND, bool SHARE>
__device__ __forceinline__ void pass_block(const PassArgs& a, int block) {
    // [warp][row][64] sums, [warp][row][4] reference, sum and unit, [row] owner, [warp] ring
    extern __shared__ __align__(128) float smem[];  // KeyCopy places rows of the rings by their address bits
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    // Blocks with the most keys (the last rows) first.
    int split = block % a.splits, splits = a.splits;
    const int unit_blocks = (a.units + a.pack - 1) / a.pack, group = warp / a.key_warps;
    int unit = (block / a.splits) % unit_blocks * a.pack + group / a.unit_tiles;
    int row_block = a.row_blocks - 1 - block / (a.splits * unit_blocks);
    long long part0 = a.part0;
    if constexpr (SHARE) {
        pass_begin(a.beside);
        const int kvh = block % a.hkv;
        row_block = block / a.hkv % a.row_blocks;
        const int slot = block / (a.hkv * a.row_blocks);
        __shared__ Share shared_share;
        if (warp == 0) {
            const Share found = share_of(a, slot, lane);
            if (lane == 0) shared_share = found;
        }
        __syncthreads();
        const Share share = shared_share;
        if (share.parts == 0) return;
        if (threadIdx.x == 0) a.shares[share.request] = make_int2(share.first, share.parts);
        unit = share.request * a.hkv + kvh;
        split = slot - share.first;
        splits = share.parts;
        part0 += (share.first - (long long)share.request * splits) * a.rows.rows * a.hq;
    }
    const int phase = warp % a.key_warps;
    const int tile = row_block * (WARPS / a.key_warps) + group % a.unit_tiles;
    UnitRows rows(a, min(unit, a.units - 1));
    if constexpr (!SHARE) pass_begin(a.beside);  // the indices above are computed while the kernel before ends
    rows.locate();
    const int e0 = tile * ROWS;
    const bool any_row = unit < a.units && group < a.pack * a.unit_tiles && e0 < rows.size();
    if (any_row) rows.tile(e0, ROWS);
    const KeyRange& r = rows.keys;
    int hi, lo;  // keys of the lane's row, g
    const int row_of = any_row ? rows.pair(e0 + g, lo, hi) : -1;

    // Sums of the rows in shared memory: the matrix unit drops the bits of a sum
    // that its 24 do not hold (it does not round them), so a long chain of products drifts towards
    // zero: 256 key tiles in one chain were 4e-6 off. Every FOLD tiles the registers are added here.
    float4* const acc = reinterpret_cast<float4*>(smem + (warp * ROWS + g) * 64 + 16 * t);
    // See kv8_move; no lift, and extra is the factor of the value scales. A row's first off is above this one, so that
    // the factor for what was there (nothing) is 0.
    float off = KV8_REF_NONE, extra = 0.f, sum = 0.f;  // extra 0: KV8_UNSET
    bool set = false;                                  // all rows of the warp have
    float o[8][4];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][j] = 0.f;
    };
    clear();
    auto fold = [&](bool first) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float4 y = first ? make_float4(0.f, 0.f, 0.f, 0.f) : acc[j];
            auto add = [&](float& x, int d) {
                const float* const from = o[4 * (j & 1) + d] + (j >> 1);
                const float v = from[0] + from[2];  // the planes
                x = first ? v : x + v;
            };
            add(y.x, 0); add(y.y, 1); add(y.z, 2); add(y.w, 3);
            acc[j] = y;
        }
    };

    const int t0 = r.lo >> 4, tiles = any_row ? (r.hi >> 4) - t0 + 1 : 0;
    const int per = max((tiles + splits - 1) / splits, 2 * a.key_warps);  // a short request in fewer parts
    const int end = min(tiles, (split + 1) * per);
    int at = split * per + phase;
    bool folded = false;
    if (at < end) {
        const bool l1 = a.key_warps == 1;  // the block's warps read the same keys
        const uint8_t* const ring = reinterpret_cast<const uint8_t*>(smem) + SUM_BYTES + warp * RING * TILE_BYTES;
        // The queries' loads go first: they are back when the first key tiles are.
        float x[16];
        if (row_of >= 0) {
            const int row = row_of / a.hq, head = row_of - row * a.hq;
            const float* src = a.q + (size_t)row * a.ldq + (size_t)head * 64 + 16 * t;
            if (a.qvec) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 f = reinterpret_cast<const float4*>(src)[j];
                    x[4 * j] = f.x; x[4 * j + 1] = f.y; x[4 * j + 2] = f.z; x[4 * j + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) x[j] = src[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = 0.f;
        }
        const KeyCopy copy(a.c, r, smem_u32(ring), lane, l1);
#pragma unroll
        for (int i = 0; i < RING - 1; i++) {
            if (at + i * a.key_warps < end) copy.tile(r, (t0 + at + i * a.key_warps) * 16, i, lane);
            copies_commit();
        }
        // Queries: 16 dimensions of the lane's row, as fp16 planes of a power-of-two multiple.
        uint32_t qa[4][4];
        float q_scale;
        {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < 16; j++) top = fmaxf(top, fabsf(x[j]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float up = power_to(top, 13);
            q_scale = 0.125f * 1.4426950408889634f / up;  // scores in powers of two
#pragma unroll
            for (int s = 0; s < 4; s++) {
                split_half2(x[4 * s] * up, x[4 * s + 1] * up, qa[s][0], qa[s][1]);
                split_half2(x[4 * s + 2] * up, x[4 * s + 3] * up, qa[s][2], qa[s][3]);
            }
        }

        int chain = 0;
        for (int stage = 0; at < end; at += a.key_warps, stage = (stage + 1) & (RING - 1)) {
            if (++chain == FOLD + 1) {
                fold(!folded);
                clear();
                folded = true;
                chain = 1;
            }
            const int u0 = (t0 + at) * 16;
            __syncwarp();  // every lane has read the tile that is copied over
            if (at + (RING - 1) * a.key_warps < end)
                copy.tile(r, u0 + 16 * (RING - 1) * a.key_warps, (stage + RING - 1) & (RING - 1), lane);
            copies_commit();
            copies_wait<RING - 1>();
            __syncwarp();
            const uint8_t* const x = ring + stage * TILE_BYTES;
            const float4 ks4 = *reinterpret_cast<const float4*>(x + 2048 + 16 * t), vs4 = *reinterpret_cast<const float4*>(x + 2112 + 16 * t);
            // The scales of key and query first: their product is of a score's size, while a sum of codes
            // times a large key scale may be infinite.
            const float ks[4] = {ks4.x * q_scale, ks4.y * q_scale, ks4.z * q_scale, ks4.w * q_scale};
            float vs[4] = {vs4.x, vs4.y, vs4.z, vs4.w};

            // Scores before scaling: 4 keys of the lane's row.
            float s[4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint4 k = *reinterpret_cast<const uint4*>(x + (4 * (g >> 1) + 2 * j + (g & 1)) * 64 + 16 * t);
                const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    uint32_t b0, b1;
                    to_half<KIND>(kw[w], b0, b1);
                    mma16816(c, qa[w], b0, b1);
                }
                s[2 * j] = c[0] + c[2];
                s[2 * j + 1] = c[1] + c[3];
            }
            const bool whole = u0 >= r.in_lo && u0 + 15 <= r.in_hi;
#pragma unroll
            for (int k = 0; k < 4; k++) vs[k] *= extra;  // may be infinite: the product with a weight is then too, or NaN
            // Weights 2^(score - off), times the value rows' scales.
            float w[4], add;
            auto weigh = [&](auto masked, auto slow, float after) {
                float p[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    p[k] = ex2(slow ? kv8_score(s[k], ks[k]) - off : fmaf(s[k], ks[k], -off));
                    w[k] = p[k] * vs[k] * after;
                    if (masked) {
                        const bool on = u0 + 4 * t + k >= lo && u0 + 4 * t + k <= hi;
                        p[k] = on ? p[k] : 0.f;
                        w[k] = on ? w[k] : 0.f;  // a scale of a key that this row does not see may be NaN
                    }
                }
                add = (p[0] + p[1]) + (p[2] + p[3]);
                return (fabsf(w[0]) + fabsf(w[1])) + (fabsf(w[2]) + fabsf(w[3])) <= KV8_PRODUCT_MAX && add <= KV8_WEIGHT_MAX;
            };
            bool fine = false;
            if (set) fine = whole ? weigh(std::false_type{}, std::false_type{}, 1.f) : weigh(std::true_type{}, std::false_type{}, 1.f);
            if (__any_sync(0xffffffffu, !fine)) {  // rare: a row's units are set, or move
                float z[4], v[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    vs[k] = reinterpret_cast<const volatile float*>(x + 2112 + 16 * t)[k];  // as they are (read again: registers)
                    const bool on = whole || (u0 + 4 * t + k >= lo && u0 + 4 * t + k <= hi);
                    z[k] = on ? kv8_score(s[k], ks[k]) : -INFINITY;
                    v[k] = on ? fabsf(vs[k]) : 0.f;
                }
                float total = extra == 0.f ? KV8_UNSET : (float)((int)(__float_as_uint(extra) >> 23) - 127);
                const Kv8Move move = kv8_move(z, v, off, total, [](float) { return 0.f; });
                extra = total == KV8_UNSET ? 0.f : kv8_power(total);
                if (move.sums != 1.f || move.outputs != 1.f) {
                    const float f = move.outputs;
                    sum *= move.sums;
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        o[n][0] *= f; o[n][1] *= f; o[n][2] *= f; o[n][3] *= f;
                    }
                    if (folded) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float4 y = acc[j];
                            acc[j] = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
                        }
                    }
                }
                set = __all_sync(0xffffffffu, extra != 0.f);
                weigh(std::true_type{}, std::true_type{}, extra);
            }
            uint32_t pa[4];
            sum += add;
            split_half2(w[0], w[1], pa[0], pa[1]);
            split_half2(w[2], w[3], pa[2], pa[3]);
            // Values: dimensions 8g .. 8g+7 of keys 4t .. 4t+3, the two keys of a pair side by side.
            uint2 v[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                v[i] = *reinterpret_cast<const uint2*>(x + 1024 + ((4 * t + i) ^ (t & 1)) * 64 + 16 * ((g >> 1) ^ (t & 2)) + 8 * (g & 1));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t v0 = h ? v[0].y : v[0].x, v1 = h ? v[1].y : v[1].x;
                const uint32_t v2 = h ? v[2].y : v[2].x, v3 = h ? v[3].y : v[3].x;
                uint32_t b0[4], b1[4];
                to_half<KIND>(__byte_perm(v0, v1, 0x5140), b0[0], b0[1]);
                to_half<KIND>(__byte_perm(v0, v1, 0x7362), b0[2], b0[3]);
                to_half<KIND>(__byte_perm(v2, v3, 0x5140), b1[0], b1[1]);
                to_half<KIND>(__byte_perm(v2, v3, 0x7362), b1[2], b1[3]);
#pragma unroll
                for (int d = 0; d < 4; d++) mma16816(o[4 * h + d], pa, b0[d], b1[d]);
            }
        }
    }

    // Merge the key_warps warps of each row tile.
    fold(!folded);
    float4* const ml = reinterpret_cast<float4*>(smem + WARPS * ROWS * 64);  // reference, sum; see OverSum
    int* const owner = reinterpret_cast<int*>(ml + WARPS * ROWS);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (t == 0) {
        const float2 all = kv8_total(off, sum);
        const OverSum out(extra == 0.f ? 1.f : extra, sum);
        ml[warp * ROWS + g] = make_float4(all.x, all.y, out.first, out.second);
        if (phase == 0) owner[group * ROWS + g] = row_of;
    }
    __syncthreads();
    const int rows_here = WARPS / a.key_warps * ROWS;
    for (int e = threadIdx.x; e < rows_here * 16; e += WARPS * 32) {
        const int row = e >> 4, d4 = e & 15, target = owner[row];
        if (target < 0) continue;
        const int base = row / ROWS * a.key_warps * ROWS + row % ROWS;
        float4 m[WARPS], v[WARPS];  // all loads before the first use
        float top = KV8_REF_NONE, l = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
            const bool on = k < a.key_warps;
            m[k] = on ? ml[base + k * ROWS] : make_float4(KV8_REF_NONE, 0.f, 0.f, 0.f);
            v[k] = on ? reinterpret_cast<const float4*>(smem + (base + k * ROWS) * 64)[d4] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < WARPS; k++) top = fmaxf(top, m[k].x);
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
            m[k].y *= ex2(m[k].x - top);
            l += m[k].y;
        }
        const float over = rcp(l);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
            const float f = m[k].y * over;
            y.x += f * (v[k].x * m[k].z * m[k].w); y.y += f * (v[k].y * m[k].z * m[k].w);
            y.z += f * (v[k].z * m[k].z * m[k].w); y.w += f * (v[k].w * m[k].z * m[k].w);
        }
        if (!a.parted) {
            const int qrow = target / a.hq, head = target - qrow * a.hq;
            float* dst = a.out + (size_t)qrow * a.ldo + (size_t)head * 64 + 4 * d4;
            if (a.ovec) {
                *reinterpret_cast<float4*>(dst) = y;
            } else {
                dst[0] = y.x; dst[1] = y.y; dst[2] = y.z; dst[3] = y.w;
            }
        } else {
            const long long part = part0 + (long long)target * splits + split;
            if (d4 == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(top, l);
            if (!(l == 0.f)) reinterpret_cast<float4*>(a.part_o + part * 64)[d4] = y;  // else not read
        }
    }
}

template <int KIND, bool SHARE>
__global__ void __launch_bounds__(WARPS * 32, 2) kv8_pass_kernel(const PassArgs a) {
    pass_block<KIND, SHARE>(a, blockIdx.x);
    if (a.beside) pdl_wait();
}

// The two passes of a call behind a prefix in one launch.
template <int PREFIX_KIND, int KIND>
__global__ void __launch_bounds__(WARPS * 32, 2) kv8_passes_kernel(const PassArgs prefix, const PassArgs own, int prefix_blocks) {
    const int block = blockIdx.x;
    if (block < prefix_blocks) pass_block<PREFIX_KIND, false>(prefix, block);
    else pass_block<KIND, false>(own, block - prefix_blocks);
}

// Joins the parts of each (row, head): out = sum_s w_s O_s, w_s = 2^(m_s - M) l_s / (the sum of these). A
// block a (row, head): a thread a part for the weights; 16 lanes cover the 64 dimensions, the 8 groups of 16
// take parts in turn, so that 64 parts are one round trip to memory, begun before the weights are known.
struct JoinArgs {
    Kv8Rows rows;
    int hq, splits, prefix_splits;  // parts of a request's own pass (shares: by request) and of the prefix's
    const int2* shares;
    long long own0;                 // first part of the own pass, behind the prefix's
    const float *part_o, *part_ml;
    float* out; int ldo; bool ovec;
};
constexpr int JOIN_THREADS = 128, JOIN_GROUPS = JOIN_THREADS / 16, JOIN_AHEAD = 8;
constexpr int MOST_SPLITS = 512;  // of a pass

__global__ void __launch_bounds__(JOIN_THREADS) kv8_join_kernel(const JoinArgs a) {
    __shared__ float2 weight[2 * MOST_SPLITS];  // (reference, sum), then (weight, -)
    __shared__ float warp_top[JOIN_THREADS / 32], warp_sum[JOIN_THREADS / 32];
    __shared__ float4 partial[JOIN_THREADS / 32][16];
    const int group = threadIdx.x >> 4, d4 = threadIdx.x & 15, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x / a.hq, request = row / a.rows.rows;
    pdl_wait();
    pdl_launch();
    if (row - request * a.rows.rows >= kv8_span(a.rows, request).count) return;
    const int2 own = a.shares ? a.shares[request] : make_int2(request * a.splits, a.splits);
    const int parts = a.prefix_splits + own.y;
    const long long size = (long long)a.rows.rows * a.hq;
    const long long prefix_at = (long long)blockIdx.x * a.prefix_splits;
    const long long own_at = a.own0 + (own.x - (long long)request * own.y) * size + (long long)blockIdx.x * own.y - a.prefix_splits;
    auto at = [&](int s) { return (s < a.prefix_splits ? prefix_at : own_at) + s; };
    auto output = [&](int s) { return reinterpret_cast<const float4*>(a.part_o)[at(s) * 16 + d4]; };
    float4 ahead[JOIN_AHEAD];
#pragma unroll
    for (int i = 0; i < JOIN_AHEAD; i++)
        ahead[i] = group + i * JOIN_GROUPS < parts ? output(group + i * JOIN_GROUPS) : make_float4(0.f, 0.f, 0.f, 0.f);
    float top = KV8_REF_NONE, sum = 0.f;
    for (int s = threadIdx.x; s < parts; s += JOIN_THREADS) {
        const float2 p = reinterpret_cast<const float2*>(a.part_ml)[at(s)];
        weight[s] = p;
        top = fmaxf(top, p.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(warp_top[0], warp_top[1]), fmaxf(warp_top[2], warp_top[3]));
    for (int s = threadIdx.x; s < parts; s += JOIN_THREADS) {
        const float2 p = weight[s];
        const float w = ex2(p.x - top) * p.y;
        sum += w;
        weight[s].x = p.y == 0.f ? -1.f : w;  // a part without a key has no outputs
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    const float over = rcp((warp_sum[0] + warp_sum[1]) + (warp_sum[2] + warp_sum[3]));
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int s, const float4& v) {
        const float w = weight[s].x, f = w * over;
        if (w < 0.f) return;
        y.x += f * v.x; y.y += f * v.y; y.z += f * v.z; y.w += f * v.w;
    };
#pragma unroll
    for (int i = 0; i < JOIN_AHEAD; i++) {
        if (group + i * JOIN_GROUPS < parts) add(group + i * JOIN_GROUPS, ahead[i]);
    }
#pragma unroll 4
    for (int s = group + JOIN_AHEAD * JOIN_GROUPS; s < parts; s += JOIN_GROUPS) add(s, output(s));
    y.x += __shfl_xor_sync(0xffffffffu, y.x, 16);
    y.y += __shfl_xor_sync(0xffffffffu, y.y, 16);
    y.z += __shfl_xor_sync(0xffffffffu, y.z, 16);
    y.w += __shfl_xor_sync(0xffffffffu, y.w, 16);
    if (lane < 16) partial[warp][d4] = y;
    __syncthreads();
    if (threadIdx.x >= 16) return;
    const float4 p0 = partial[0][d4], p1 = partial[1][d4], p2 = partial[2][d4], p3 = partial[3][d4];
    y = make_float4((p0.x + p1.x) + (p2.x + p3.x), (p0.y + p1.y) + (p2.y + p3.y), (p0.z + p1.z) + (p2.z + p3.z),
                    (p0.w + p1.w) + (p2.w + p3.w));
    float* dst = a.out + (size_t)row * a.ldo + (size_t)(blockIdx.x - row * a.hq) * 64 + 4 * d4;
    if (a.ovec) {
        *reinterpret_cast<float4*>(dst) = y;
    } else {
        dst[0] = y.x; dst[1] = y.y; dst[2] = y.z; dst[3] = y.w;
    }
}

// The same for at most JOIN_GROUPS parts: a group of 16 lanes a (row, head), every lane all weights. The
// reductions over a block above take 0.5 us longer.
__global__ void __launch_bounds__(JOIN_THREADS) kv8_join_few_kernel(const JoinArgs a, int pairs) {
    const int pair = blockIdx.x * JOIN_GROUPS + (threadIdx.x >> 4), d4 = threadIdx.x & 15;
    const int row = pair / a.hq, request = row / a.rows.rows;
    pdl_wait();
    pdl_launch();
    if (pair >= pairs) return;
    if (row - request * a.rows.rows >= kv8_span(a.rows, request).count) return;
    const long long prefix_at = (long long)pair * a.prefix_splits, own_at = a.own0 + (long long)pair * a.splits - a.prefix_splits;
    const int parts = a.prefix_splits + a.splits;
    float2 p[JOIN_GROUPS];
    float4 v[JOIN_GROUPS];
    float top = KV8_REF_NONE, sum = 0.f;
#pragma unroll
    for (int s = 0; s < JOIN_GROUPS; s++) {
        const long long at = (s < a.prefix_splits ? prefix_at : own_at) + s;
        p[s] = make_float2(KV8_REF_NONE, 0.f);
        if (s < parts) {
            p[s] = reinterpret_cast<const float2*>(a.part_ml)[at];
            v[s] = reinterpret_cast<const float4*>(a.part_o)[at * 16 + d4];
        }
    }
#pragma unroll
    for (int s = 0; s < JOIN_GROUPS; s++) top = fmaxf(top, p[s].x);
#pragma unroll
    for (int s = 0; s < JOIN_GROUPS; s++) {
        p[s].x = ex2(p[s].x - top) * p[s].y;
        sum += p[s].x;
    }
    const float over = rcp(sum);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < JOIN_GROUPS; s++) {
        if (p[s].y == 0.f) continue;  // a part without a key has no outputs
        const float f = p[s].x * over;
        y.x += f * v[s].x; y.y += f * v[s].y; y.z += f * v[s].z; y.w += f * v[s].w;
    }
    float* dst = a.out + (size_t)row * a.ldo + (size_t)(pair - row * a.hq) * 64 + 4 * d4;
    if (a.ovec) {
        *reinterpret_cast<float4*>(dst) = y;
    } else {
        dst[0] = y.x; dst[1] = y.y; dst[2] = y.z; dst[3] = y.w;
    }
}

Kv8View view(const mt_kv8_cache* c) {
    return Kv8View{c->k, c->v, c->k_scale, c->v_scale, c->request_stride, c->capacity, c->kind};
}

// How a pass is laid out over the GPU.
struct PassPlan {
    bool wide;
    int units, row_blocks, key_warps, pack, unit_tiles, splits, chunk, slots;
};

// `units` row spaces of `qrows` (row, head) rows each over at most `keys` keys, `requests` of them of
// lengths that may differ; the first row sees `unseen` fewer keys than the last.
PassPlan plan_pass(int sm_count, long long units, int requests, long long qrows, int keys, int unseen) {
    PassPlan p{};
    if (units < 1) return p;
    // Which kernel: by their estimated times, in ns. The warp kernel takes 5 ps a (row, head) pair and key that
    // it sees, once the GPU is full; a wide block takes 14 us to start and finish, 2.2 us for 64 keys (1.4 us
    // with up to 128 rows), and a later one on the same SM another 8 us. Measured in us, wide against warp
    // kernel, one call behind the other in a graph (int8, 14 heads on 2 unless said): one request of 16 rows over
    // 300 keys 12.7 / 5.2, 16 over 4000 17.7 / 11.2, 512 over themselves 22.3 / 19.8, 37 over 4000 22.5 / 14.3,
    // 64 over 4000 22.7 / 22.0; 8 requests of 8 rows over 4000 24.2 / 25.8, of 64 rows over 1000 24.3 / 36.8;
    // 64 requests of 8 rows over 400 keys 21.4 / 18.6, of 16 rows 22.8 / 33.4; 11 requests of 113 rows over 350,
    // 16 heads on 16, 39.2 / 42.1; a prefix of 9000 for 32 requests 24.0 / 21.9, for 414 rows 73.7 / 289. With a
    // window the estimate counts keys that rows do not see: 700 rows over 1 18.1 / 8.9, 400 over 65 20.1 / 8.6,
    // 4096 over 512 71.8 / 141, all of them wide. Its keys are split over
    // the SMs that its blocks leave free, two tiles a part or more (four: 64 rows over 4000 keys 24.0).
    {
        const long long row_blocks = (qrows + KV8_WIDE_ROWS - 1) / KV8_WIDE_ROWS, blocks = units * row_blocks;
        const long long tiles = (keys + 15 + KV8_WIDE_KEYS - 1) / KV8_WIDE_KEYS;
        long long s = (sm_count < MOST_SPLITS ? sm_count : MOST_SPLITS) / blocks;
        if (s > tiles / 2) s = tiles / 2;
        if (s < 1) s = 1;
        const long long chunk = (tiles + s - 1) / s, waves = (blocks * s + sm_count - 1) / sm_count;
        const long long each = blocks * tiles / sm_count;
        const double tile = qrows <= KV8_WIDE_ROWS / 2 ? 1.4e3 : 2.2e3;
        const double wide = 14e3 + 8e3 * (double)(waves - 1) + tile * (double)(each > chunk ? each : chunk);
        const double warp = 6e3 + 5e-3 * (double)units * (double)qrows * ((double)keys - 0.5 * unseen);
        if (wide < warp) {
            p.wide = true;
            p.units = (int)units;
            p.row_blocks = (int)row_blocks;
            p.chunk = (int)chunk;
            p.splits = (int)((tiles + chunk - 1) / chunk);
            return p;
        }
    }
    const int key_tiles = (keys + 15) / 16 + 1;
    const long long row_tiles = (qrows + ROWS - 1) / ROWS;
    // Warps of a block: over the keys of one row tile, unless that makes more blocks than are resident at once
    // or there are not that many key tiles; then over row tiles, of several units where one has too few.
    auto pack_at = [&](int kw) { return row_tiles < WARPS / kw ? (int)(WARPS / kw / row_tiles) : 1; };
    auto blocks_at = [&](int kw) {
        const int pack = pack_at(kw);
        return pack > 1 ? (units + pack - 1) / pack : units * ((row_tiles + WARPS / kw - 1) / (WARPS / kw));
    };
    p.key_warps = WARPS;
    while (p.key_warps > 1 && (blocks_at(p.key_warps) > 2ll * sm_count || p.key_warps > key_tiles)) p.key_warps /= 2;
    p.units = (int)units;
    p.pack = pack_at(p.key_warps);
    p.unit_tiles = p.pack > 1 ? (int)row_tiles : WARPS;
    const long long blocks = blocks_at(p.key_warps);
    p.row_blocks = p.pack > 1 ? 1 : (int)(blocks / units);
    // Split the keys over as many blocks as are resident at once, while every warp keeps 4 tiles.
    long long s = 2ll * sm_count / blocks;
    const long long most = key_tiles / (4 * p.key_warps);
    if (s > most) s = most;
    if (s > MOST_SPLITS) s = MOST_SPLITS;
    p.splits = s < 1 ? 1 : (int)s;
    // Slots by length where a warp's walk over the longest request would be 10 tiles or more: sharing them out
    // takes 0.8 us for 8 requests, 1.5 us for 64.
    const long long slots = 2ll * sm_count * requests / blocks;
    if (p.splits > 1 && p.pack == 1 && requests > 1 && requests <= 32 * SHARE_LANES && slots > requests &&
        slots <= MOST_SPLITS && keys <= 1 << 24 && key_tiles >= 10ll * p.key_warps * p.splits)
        p.slots = (int)(slots < most * requests ? slots : most * requests);
    return p;
}

struct Plan {
    PassPlan own, prefix;
    long long own0, parts;  // first part of the own pass, all parts; 0 parts: written out at once
    size_t o_bytes, ml_bytes, bytes;
};

// The sizes that make_plan is for, and that attention() accepts.
bool plannable(int prefix_len, const mt_kv8_cache* cache, int requests, int rows, int hq, int window) {
    return cache && prefix_len >= 0 && prefix_len <= 1 << 30 && requests > 0 && rows > 0 && hq > 0 && hq <= 1024 && cache->kv_heads > 0 &&
           hq % cache->kv_heads == 0 && cache->capacity > 0 && cache->capacity <= 1 << 30 && window >= 0 && rows <= cache->capacity &&
           (window == 0 || (long long)window + rows - 1 <= cache->capacity) && (long long)requests * rows <= 0x7FFFFF00ll / hq;
}

Plan make_plan(const mt_ctx* ctx, int prefix_len, const mt_kv8_cache* cache, int requests, int rows, int hq, int window) {
    Plan p{};
    const int hkv = cache->kv_heads;
    const long long group = hq / hkv;
    const long long seen = window > 0 ? (long long)window + rows - 1 : cache->capacity;
    const long long size = (long long)rows * hq;
    const int keys = (int)(seen < cache->capacity ? seen : cache->capacity);
    p.own = plan_pass(ctx->sm_count, (long long)requests * hkv, requests, rows * group, keys, window > 0 ? 0 : rows - 1);
    if (prefix_len > 0) {
        p.prefix = plan_pass(ctx->sm_count, hkv, 1, (long long)requests * rows * group, prefix_len, 0);
        p.own0 = (long long)p.prefix.splits * requests * size;
    }
    if (prefix_len > 0 || p.own.splits > 1 || p.own.slots > 0) {
        p.parts = p.own0 + (p.own.slots > 0 ? p.own.slots : (long long)requests * p.own.splits) * size;
        p.o_bytes = (size_t)p.parts * 64 * sizeof(float);
        p.ml_bytes = (size_t)p.parts * 2 * sizeof(float);
        p.bytes = p.o_bytes + p.ml_bytes + (p.own.slots > 0 ? requests * sizeof(int2) : 0);
    }
    return p;
}

unsigned pass_blocks(const PassArgs& a) {
    return (unsigned)(a.slots > 0 ? a.slots * a.hkv * a.row_blocks : (a.units + a.pack - 1) / a.pack * a.row_blocks * a.splits);
}

template <typename... Params, typename... Args>
void launch_warps(void (*kernel)(Params...), PerDeviceOnce& once, unsigned blocks, cudaStream_t s, const Args&... args) {
    once([kernel] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
    launch_k(kernel, dim3(blocks), WARPS * 32, SMEM, s, args...);
}

template <int KIND, bool SHARE>
void launch_pass_as(const PassArgs& a, cudaStream_t s) {
    static PerDeviceOnce once;
    launch_warps(kv8_pass_kernel<KIND, SHARE>, once, pass_blocks(a), s, a);
}

void launch_pass(const PassArgs& a, cudaStream_t s) {
    if (a.c.kind == MT_KV_INT8) a.slots > 0 ? launch_pass_as<MT_KV_INT8, true>(a, s) : launch_pass_as<MT_KV_INT8, false>(a, s);
    else a.slots > 0 ? launch_pass_as<MT_KV_E4M3, true>(a, s) : launch_pass_as<MT_KV_E4M3, false>(a, s);
}

template <int PREFIX_KIND, int KIND>
void launch_passes_as(const PassArgs& prefix, const PassArgs& own, cudaStream_t s) {
    static PerDeviceOnce once;
    launch_warps(kv8_passes_kernel<PREFIX_KIND, KIND>, once, pass_blocks(prefix) + pass_blocks(own), s, prefix, own, (int)pass_blocks(prefix));
}

void launch_passes(const PassArgs& prefix, const PassArgs& own, cudaStream_t s) {
    if (prefix.c.kind == MT_KV_INT8)
        own.c.kind == MT_KV_INT8 ? launch_passes_as<MT_KV_INT8, MT_KV_INT8>(prefix, own, s) : launch_passes_as<MT_KV_INT8, MT_KV_E4M3>(prefix, own, s);
    else
        own.c.kind == MT_KV_INT8 ? launch_passes_as<MT_KV_E4M3, MT_KV_INT8>(prefix, own, s) : launch_passes_as<MT_KV_E4M3, MT_KV_E4M3>(prefix, own, s);
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
    MT_REQUIRE(ctx, (long long)requests * rows * hq <= 0x7FFFFF00ll, MT_ERR_SHAPE, "%s: %d requests of %d rows of %d heads",
               what, requests, rows, hq);
    if (requests == 0 || rows == 0) return MT_OK;
    const Plan plan = make_plan(ctx, prefix_len, cache, requests, rows, hq, window);
    MT_REQUIRE(ctx, plan.bytes == 0 || (workspace && have >= plan.bytes && ((uintptr_t)workspace & 15u) == 0), MT_ERR_CAPACITY,
               "%s: workspace of %zu bytes (16-byte aligned), needs %zu", what, workspace ? have : (size_t)0, plan.bytes);
    DeviceGuard guard(ctx->device);
    MT_REQUIRE(ctx, guard.err == cudaSuccess, MT_ERR_CUDA, "%s: %s", what, cudaGetErrorString(guard.err));
    cudaStream_t s = as_stream(stream);
    PassArgs a{};
    a.q = q; a.ldq = ldq; a.qvec = ((uintptr_t)q & 15u) == 0 && ldq % 4 == 0;
    a.out = out; a.ldo = ldo; a.ovec = ((uintptr_t)out & 15u) == 0 && ldo % 4 == 0;
    a.rows = Kv8Rows{positions, counts, rows, cache->base};
    a.requests = requests; a.hq = hq; a.hkv = hkv; a.group = hq / hkv;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + plan.o_bytes / sizeof(float);
    int2* const shares = reinterpret_cast<int2*>(static_cast<char*>(workspace) + plan.o_bytes + plan.ml_bytes);
    a.parted = plan.parts > 0;
    auto lay_out = [&](const PassPlan& p) {
        a.units = p.units; a.row_blocks = p.row_blocks; a.splits = p.splits; a.key_warps = p.key_warps;
        a.pack = p.pack; a.unit_tiles = p.unit_tiles;
        a.slots = p.slots; a.shares = shares;
    };
    auto run = [&](const PassPlan& p) {
        if (p.wide) launch_kv8_wide(a, p.chunk, ctx->d_status, s);
        else launch_pass(a, s);
    };
    const long long size = (long long)rows * hq;
    const bool together = prefix_len > 0 && !plan.prefix.wide && !plan.own.wide && plan.own.slots == 0;
    PassArgs before{};
    if (prefix_len > 0) {
        lay_out(plan.prefix);
        a.c = view(prefix); a.prefix_len = prefix_len; a.part0 = 0;
        if (together) before = a;
        else run(plan.prefix);
    }
    lay_out(plan.own);
    a.c = view(cache); a.prefix_len = 0; a.part0 = plan.own0; a.window = window;
    a.beside = prefix_len > 0 && !together;
    if (together) launch_passes(before, a, s);
    else run(plan.own);
    if (a.parted) {
        const JoinArgs j{a.rows, hq, plan.own.splits, plan.prefix.splits, plan.own.slots > 0 ? shares : nullptr,
                         plan.own0, a.part_o, a.part_ml, out, ldo, a.ovec};
        const unsigned pairs = (unsigned)(requests * size);
        if (!j.shares && j.splits + j.prefix_splits <= JOIN_GROUPS)
            launch_k(kv8_join_few_kernel, dim3((pairs + JOIN_GROUPS - 1) / JOIN_GROUPS), JOIN_THREADS, 0, s, j, (int)pairs);
        else
            launch_k(kv8_join_kernel, dim3(pairs), JOIN_THREADS, 0, s, j);
    }
    return check_launch(ctx, what);
}

}  // namespace

}  // namespace mt

using namespace mt;

extern "C" {

size_t mt_attention_kv8_workspace(const mt_ctx* ctx, const mt_kv8_cache* cache, int requests, int rows, int hq, int window) {
    return ctx && plannable(0, cache, requests, rows, hq, window) ? make_plan(ctx, 0, cache, requests, rows, hq, window).bytes : 0;
}

size_t mt_attention_prefix_kv8_workspace(const mt_ctx* ctx, int prefix_len, const mt_kv8_cache* cache, int requests,
                                         int rows, int hq) {
    return ctx && plannable(prefix_len, cache, requests, rows, hq, 0) ? make_plan(ctx, prefix_len, cache, requests, rows, hq, 0).bytes : 0;
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
