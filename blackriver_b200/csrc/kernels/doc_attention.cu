// Attention over packed documents, forward and backward, fp16 on the tcgen05 tensor cores.
//
//   x_ij = q_i . k_j / sqrt(d)        s_ij = cap tanh(x_ij / cap)  (cap > 0)        s_ij -= slope_h |i - j|  (slopes given)
//   P = softmax over the keys lo_i <= j < hi_i,     O = P V,     a query without a key: O = 0, lse = 0
//   dS = P (dO V^T - delta) (1 - tanh^2),  delta_i = dO_i . O_i;   dQ = dS K / sqrt(d),  dK = dS^T Q / sqrt(d),  dV = P^T dO
//
// A token's spans say which keys it sees as a query and which queries see it as a key; inside a row of the batch both
// bounds of both spans never fall from one token to the next (documents follow one another), so the keys that a tile of
// queries needs lie between its first token's lo and its last token's hi, and blocks outside are never touched: the
// work grows with the documents' lengths, not with the row's.  Query heads h*g .. share a key head when there are fewer.
//
// What is masked may hold anything.  A masked score or gradient is replaced, never multiplied.  A masked value row still
// meets a probability of zero inside the tensor core, and 0 * NaN is NaN; the epilogues notice an accumulator that is not
// finite, and a row that sees nothing of the kind itself is evaluated again in fp32 over its visible pairs alone.  So a NaN
// or an infinity reaches exactly the rows that see it, and costs nothing where there is none.
//
// Every mbarrier wait is bounded (see brk_ptx.cuh); a give-up raises g_doc_error.
#include <atomic>
#include <type_traits>

#include "brk_attn.cuh"
#include "brk_common.cuh"
#include "brk_ptx.cuh"

namespace brk {

using namespace ptx;

__device__ int g_doc_error = 0;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int DA_THREADS = 64 + 512;        // producer warp, MMA warp, sixteen row-owner warps
constexpr int DA_SORT = 512;                // tiles whose order a CTA sorts; more are taken as they come

struct DocAttn {
    const __half *q, *k, *v;
    const int4* spans;                      // [batch, tokens]: lo, hi, qlo, qhi
    const float* slopes;                    // [heads] or null
    int64_t ld_q, ld_kv, ld_out;
    int batch, tokens, heads, kv_heads;
    float scale, scale_log2;                // 1/sqrt(d), times log2(e)
    float cap_log2, cap_in;                 // cap log2(e); 1 / (sqrt(d) cap)
    float cap_curve;                        // -1 / cap_log2^2: the tanh's derivative is 1 + cap_curve s^2 of the capped score s
    float cap_poly[5];                      // coefficients of the capped score, see da_capped_near
    // forward
    __half* out;
    float* lse;                             // [batch, heads, tokens], natural log
    // backward
    const __half* d_out;
    const float* lse_in;
    const float* delta;                     // [batch, heads, tokens]
    __half *dq, *dk, *dv;
    int64_t ld_dq, ld_dkv;
};

// ---- scores --------------------------------------------------------------------------------------------------------------

// The cap.  tanh(u) for |u| <= 0.6 is an odd polynomial (least maximum relative error over the interval, 1.8e-7 in fp32) on
// the FMA units, two scores at a time.  Wider arguments take 1 - 2 / (1 + e^2u), two operations on the special function unit,
// of which the softmax already needs one per score: at 16 a clock and SM that unit, not the tensor core, would set the
// pace.  Both are within 2e-7 of tanh relative to it, 1e-5 of the exponent at a cap of 50; the hardware tanh's 2^-11 would be
// 0.02 of it.  A reach of 0.75 would need a sixth term for that.
constexpr float TANH_REACH = 0.6f;
constexpr float TANH_1 = 0.99999994f, TANH_3 = -0.33332309f, TANH_5 = 0.13310173f, TANH_7 = -0.052101482f, TANH_9 = 0.015475427f;
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float da_tanh(float u) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp2(2.0f * LOG2E * u)));
    return fmaf(-2.0f, r, 1.0f);
}
// cap * tanh(raw * scale / cap) in log2 units plus `off`, by the polynomial, whose coefficients hold the cap
__device__ __forceinline__ float2 da_capped_near(float2 raw, const DocAttn& p, float2 off) {
    const float2 u = __fmul2_rn(raw, both(p.cap_in)), s = __fmul2_rn(u, u);
    float2 t = __ffma2_rn(both(p.cap_poly[4]), s, both(p.cap_poly[3]));
    t = __ffma2_rn(t, s, both(p.cap_poly[2]));
    t = __ffma2_rn(t, s, both(p.cap_poly[1]));
    t = __ffma2_rn(t, s, both(p.cap_poly[0]));
    return __ffma2_rn(t, u, off);
}
// the same without the offset for any argument
__device__ __forceinline__ float2 da_capped_far(float2 raw, const DocAttn& p) {
    const float2 u = __fmul2_rn(raw, both(p.cap_in));
    return __fmul2_rn(make_float2(da_tanh(u.x), da_tanh(u.y)), both(p.cap_log2));
}
template <bool CAP>
__device__ __forceinline__ float da_score(float raw, const DocAttn& p, float& slope_of_tanh) {
    if (!CAP) {
        slope_of_tanh = 1.0f;
        return raw * p.scale_log2;
    }
    const float t = da_tanh(raw * p.cap_in);
    slope_of_tanh = fmaf(-t, t, 1.0f);
    return t * p.cap_log2;
}
// bits [from, to) of 32, whatever lies outside of them
__device__ __forceinline__ uint32_t span_bits(int from, int to) {
    from = min(max(from, 0), 32);
    to = min(max(to, from), 32);
    return (uint32_t)((1ull << to) - (1ull << from));
}
template <bool B>
using Flag = std::integral_constant<bool, B>;
// The straight line at + slope * e over a chunk's columns, two at a time.  Four running pairs: as fused multiply-adds on the
// numbers of the columns it took a register pair for each of them.
struct Line {
    float2 v[4], step;
    __device__ __forceinline__ Line(float slope, float at) {
        const float2 first = make_float2(at, at + slope), two = both(2.0f * slope);
        v[0] = first;
#pragma unroll
        for (int i = 1; i < 4; i++) v[i] = __fadd2_rn(v[i - 1], two);
        step = both(8.0f * slope);
    }
    // columns 2i and 2i + 1; i in order
    __device__ __forceinline__ float2 next(int i) {
        const float2 r = v[i & 3];
        v[i & 3] = __fadd2_rn(r, step);
        return r;
    }
};

// ---- tiles ---------------------------------------------------------------------------------------------------------------

struct Range {
    int begin, end;
};
// a value that is the same in the whole warp, known to be
template <typename T>
__device__ __forceinline__ T uniform(T x) { return __shfl_sync(0xffffffffu, x, 0); }
// keys (KEYS) that 128 queries from t0 on see, or queries that see 128 keys, as a range of `unit`-sized blocks
template <bool KEYS>
__device__ __forceinline__ Range da_blocks(const DocAttn& p, int b, int t0, int unit) {
    Range r = {0, 0};
    if (t0 >= p.tokens) return r;
    const int4* s = p.spans + (int64_t)b * p.tokens;
    const int4 head = s[t0], tail = s[min(t0 + 127, p.tokens - 1)];
    const int lo = max(KEYS ? head.x : head.z, 0), hi = min(KEYS ? tail.y : tail.w, p.tokens);
    if (lo < hi) {
        r.begin = lo / unit;
        r.end = (hi + unit - 1) / unit;
    }
    return r;
}

// The CTAs are persistent and walk items (tile, head): tiles in the order of falling work, dealt in rounds of alternating
// direction, which evens out the totals without a counter in memory.  Every CTA sorts for itself (two loads per tile) and
// lists its items in shared memory before the walk begins: the divisions and loads behind an item cost 2000 clocks where
// a role does them between two items.  Only the items behind the list's end are worked out on the way.
constexpr int DA_LIST = 96;
struct DaItem {
    int b, t0, head, pad;
    Range r0, r1;                           // blocks that the tile's first and second half need
};
struct DaTable {
    DaItem items[DA_LIST];
    ushort4 blocks[DA_SORT];                // per tile: r0, r1
    uint16_t order[DA_SORT];
};
template <typename R>
__device__ __forceinline__ bool da_find_item(int round, int n_tiles, int n_heads, int per_row, int tile_tokens, const DaTable* table, R ranges, DaItem& m) {
    const uint32_t G = gridDim.x, c = blockIdx.x;
    const uint64_t at = (uint64_t)round * G + ((round & 1) ? G - 1 - c : c);
    if (at >= (uint64_t)n_tiles * n_heads) return false;
    const uint32_t idx = (uint32_t)at;                  // tiles times heads stay below 2^32: checked before the launch
    const int place = (int)(idx / (uint32_t)n_heads);
    m.head = (int)(idx - (uint32_t)place * n_heads);
    const bool sorted = n_tiles <= DA_SORT;
    const int tile = sorted ? table->order[place] : n_tiles - 1 - place;
    m.b = tile / per_row;
    m.t0 = (tile - m.b * per_row) * tile_tokens;
    if (sorted) {
        const ushort4 t = table->blocks[tile];
        m.r0 = {t.x, t.y};
        m.r1 = {t.z, t.w};
    } else {
        m.r0 = ranges(m.b, m.t0, false);
        m.r1 = ranges(m.b, m.t0, true);
    }
    return true;
}
// Sorts the tiles (heavier first, ties by number) and lists this CTA's items; returns how many are listed (at most DA_LIST,
// the walk goes on with da_find_item).  All threads of the CTA; ranges(b, t0, second half).
template <typename R>
__device__ __forceinline__ int da_plan_items(DaTable* table, int n_tiles, int n_heads, int per_row, int tile_tokens, R ranges) {
    if (n_tiles <= DA_SORT) {
        for (int i = threadIdx.x; i < n_tiles; i += blockDim.x) {
            const int b = i / per_row, t0 = (i - b * per_row) * tile_tokens;
            const Range x = ranges(b, t0, false), y = ranges(b, t0, true);
            table->blocks[i] = make_ushort4(x.begin, x.end, y.begin, y.end);
        }
        __syncthreads();
        auto weight = [&](int i) {
            const ushort4 t = table->blocks[i];
            return t.y - t.x + t.w - t.z;
        };
        for (int i = threadIdx.x; i < n_tiles; i += blockDim.x) {
            const int w = weight(i);
            int rank = 0;
            for (int j = 0; j < n_tiles; j++) {
                const int v = weight(j);
                rank += v > w || (v == w && j < i);
            }
            table->order[rank] = (uint16_t)i;
        }
        __syncthreads();
    }
    const uint32_t items = (uint32_t)n_tiles * n_heads;
    const uint32_t full = items / gridDim.x, rest = items - full * gridDim.x;
    // rounds this CTA has an item in: all full ones, and the last one if it is dealt that far
    const uint32_t mine = full + ((full & 1) ? (blockIdx.x >= gridDim.x - rest) : (blockIdx.x < rest));
    const int listed = (int)min(mine, (uint32_t)DA_LIST);
    for (int i = threadIdx.x; i < listed; i += blockDim.x) {
        DaItem m = {};
        da_find_item(i, n_tiles, n_heads, per_row, tile_tokens, table, ranges, m);
        table->items[i] = m;
    }
    return listed;
}

// ---- results ---------------------------------------------------------------------------------------------------------------

// one arrival for the whole warp
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void da_zero_row(__half* row, int d) {
    for (int e = 0; e < d; e += 8) *reinterpret_cast<uint4*>(row + e) = make_uint4(0, 0, 0, 0);
}
// Results leave through shared memory: a warp writes 32 rows x 32 columns into 2 KB of its own, and its first lane stores them
// with the TMA, which clips the box at the end of the row of the batch.  Stores by the owners themselves, whose neighbouring
// lanes hold rows 24 KB apart, kept the load/store unit busy for 4000 to 7000 clocks an item.
constexpr int DA_PATCH = 2048;                  // bytes a warp stages
// 16-byte piece `piece` of row `row` of a patch whose rows are COLS columns: 64-byte swizzle for 32 columns, none for 16
template <int COLS>
__device__ __forceinline__ void da_stage(unsigned char* patch, int row, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const int at = COLS == 32 ? row * 64 + ((piece ^ ((row >> 1) & 3)) << 4) : row * 32 + piece * 16;
    *reinterpret_cast<uint4*>(patch + at) = make_uint4(a, b, c, d);
}
// the warp's patch may be written again
__device__ __forceinline__ void da_patch_free() {
    if ((threadIdx.x & 31) == 0) bulk_wait_read<0>();
    __syncwarp();
}
__device__ __forceinline__ void da_patch_store(const CUtensorMap* map, const unsigned char* patch, int x, int y, int z, int tokens) {
    fence_proxy_async();
    __syncwarp();
    if ((threadIdx.x & 31) == 0 && y < tokens) {
        tma_store_3d(map, patch, x, y, z);
        bulk_commit();
    }
}
// what the warp has stored is written, so that it can be written again by plain stores
__device__ __forceinline__ void da_patch_written() {
    if ((threadIdx.x & 31) == 0) bulk_wait_all();
    __syncwarp();
}
// whether `x` holds for any thread of those that meet at the barrier
__device__ __forceinline__ bool barrier_any(int id, int threads, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.or.pred p, %2, %3, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ uint32_t da_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- rows evaluated again without the tensor core (see the top) ------------------------------------------------------------
// Called by whole warps with one row per lane, `bad` where the row's accumulator is not finite.  A row that sees an operand
// that is not finite keeps what it has (32 partners are looked at at a time, one per lane, until every bad row has found
// one); the others are evaluated one after another by the warp: a lane forms the pair terms of one partner in 32, then the
// lanes share the sum over them, D / 32 columns each.

template <int D>
__device__ __forceinline__ bool da_not_finite(const __half* row) {
    bool found = false;
    for (int c = 0; c < D; c += 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + c);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) found |= (x[e] & 0x7c00u) == 0x7c00u || (x[e] & 0x7c000000u) == 0x7c000000u;
    }
    return found;
}
template <int D>
__device__ __forceinline__ float da_dot(const __half* a, const __half* b) {
    float s = 0.0f;
    for (int c = 0; c < D; c += 8) {
        Vec<__half> x, y;
        x.load(a + c);
        y.load(b + c);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf(x.v[e], y.v[e], s);
    }
    return s;
}
// which of the bad rows see no partner for which found(partner) holds
template <typename F>
__device__ __forceinline__ uint32_t da_to_mend(bool bad, int lo, int hi, F found) {
    const int lane = threadIdx.x & 31;
    const int from = __reduce_min_sync(0xffffffffu, bad ? lo : 0x7fffffff), to = __reduce_max_sync(0xffffffffu, bad ? hi : 0);
    uint32_t left = __ballot_sync(0xffffffffu, bad);
    for (int k0 = from; k0 < to && left; k0 += 32) {
        const uint32_t hits = __ballot_sync(0xffffffffu, k0 + lane < to && found(k0 + lane));
        if (hits & span_bits(lo - k0, hi - k0)) bad = false;
        left = __ballot_sync(0xffffffffu, bad);
    }
    return left;
}
// acc[e] += w * row[lane * D / 32 + e] for each partner of a block of 32, whose weight is in the lane of its number
template <int D>
__device__ __forceinline__ void da_add_rows(float (&acc)[D / 32], float w, const __half* rows, int64_t ld, int n) {
    const int lane = threadIdx.x & 31;
    for (int i = 0; i < n; i++) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const __half2* x = reinterpret_cast<const __half2*>(rows + i * ld + lane * (D / 32));
#pragma unroll
        for (int e = 0; e < D / 64; e++) {
            const float2 f = __half22float2(x[e]);
            acc[2 * e] = fmaf(wi, f.x, acc[2 * e]);
            acc[2 * e + 1] = fmaf(wi, f.y, acc[2 * e + 1]);
        }
    }
}
template <int D>
__device__ __forceinline__ void da_store_row(__half* row, const float (&acc)[D / 32], float scale) {
    __half2* o = reinterpret_cast<__half2*>(row + (threadIdx.x & 31) * (D / 32));
#pragma unroll
    for (int e = 0; e < D / 64; e++) o[e] = __floats2half2_rn(acc[2 * e] * scale, acc[2 * e + 1] * scale);
}
// the tensors of one row of the batch and one head
template <int D>
struct DaHead {
    const __half *q, *k, *v, *g;
    const float *lse, *delta;
    float slope2;
    __device__ DaHead(const DocAttn& p, int b, int h) {
        const int64_t row = (int64_t)b * p.tokens, at = ((int64_t)b * p.heads + h) * p.tokens;
        const int kh = h / (p.heads / p.kv_heads);
        q = p.q + row * p.ld_q + h * D;
        k = p.k + row * p.ld_kv + kh * D;
        v = p.v + row * p.ld_kv + kh * D;
        g = p.d_out ? p.d_out + row * p.ld_out + h * D : nullptr;
        lse = p.lse_in ? p.lse_in + at : nullptr;
        delta = p.delta ? p.delta + at : nullptr;
        slope2 = p.slopes ? p.slopes[h] * LOG2E : 0.0f;
    }
    // score in log2 units of a visible pair
    template <bool CAP>
    __device__ float score(const DocAttn& p, int i, int j, float& dt) const {
        return da_score<CAP>(da_dot<D>(q + i * p.ld_q, k + j * p.ld_kv), p, dt) - slope2 * fabsf((float)(i - j));
    }
    // P and dS of a visible pair
    template <bool CAP>
    __device__ float pair(const DocAttn& p, int i, int j, float& ds) const {
        float dt;
        const float w = fast_exp2(score<CAP>(p, i, j, dt) - lse[i] * LOG2E);
        ds = w * (da_dot<D>(g + i * p.ld_out, v + j * p.ld_kv) - delta[i]) * dt;
        return w;
    }
};
template <int D, bool CAP>
__device__ __noinline__ void da_mend_out(const DocAttn& p, int b, int h, int i, int lo, int hi, float lse2, bool bad) {
    const DaHead<D> t(p, b, h);
    const int lane = threadIdx.x & 31;
    uint32_t left = da_to_mend(bad, lo, hi, [&](int j) { return da_not_finite<D>(t.v + j * p.ld_kv); });
    for (; left; left &= left - 1) {
        const int r = __ffs(left) - 1, ri = __shfl_sync(0xffffffffu, i, r), from = __shfl_sync(0xffffffffu, lo, r), to = __shfl_sync(0xffffffffu, hi, r);
        const float rl = __shfl_sync(0xffffffffu, lse2, r);
        float acc[D / 32] = {};
        for (int j = from; j < to; j += 32) {
            float dt, w = 0.0f;
            if (j + lane < to) w = fast_exp2(t.template score<CAP>(p, ri, j + lane, dt) - rl);
            da_add_rows<D>(acc, w, t.v + j * p.ld_kv, p.ld_kv, min(32, to - j));
        }
        da_store_row<D>(p.out + ((int64_t)b * p.tokens + ri) * p.ld_out + h * D, acc, 1.0f);
    }
}
template <int D, bool CAP>
__device__ __noinline__ void da_mend_dq(const DocAttn& p, int b, int h, int i, int lo, int hi, bool bad) {
    const DaHead<D> t(p, b, h);
    const int lane = threadIdx.x & 31;
    if (bad && (!(fabsf(t.lse[i]) < INFINITY) || !(fabsf(t.delta[i]) < INFINITY) || da_not_finite<D>(t.q + i * p.ld_q) || da_not_finite<D>(t.g + i * p.ld_out))) bad = false;
    uint32_t left = da_to_mend(bad, lo, hi, [&](int j) { return da_not_finite<D>(t.k + j * p.ld_kv) || da_not_finite<D>(t.v + j * p.ld_kv); });
    for (; left; left &= left - 1) {
        const int r = __ffs(left) - 1, ri = __shfl_sync(0xffffffffu, i, r), from = __shfl_sync(0xffffffffu, lo, r), to = __shfl_sync(0xffffffffu, hi, r);
        float acc[D / 32] = {};
        for (int j = from; j < to; j += 32) {
            float ds = 0.0f;
            if (j + lane < to) t.template pair<CAP>(p, ri, j + lane, ds);
            da_add_rows<D>(acc, ds, t.k + j * p.ld_kv, p.ld_kv, min(32, to - j));
        }
        da_store_row<D>(p.dq + ((int64_t)b * p.tokens + ri) * p.ld_dq + h * D, acc, p.scale);
    }
}
template <int D, bool CAP>
__device__ __noinline__ void da_mend_dkv(const DocAttn& p, int b, int kh, int j, int lo, int hi, bool bad) {
    const int group = p.heads / p.kv_heads, lane = threadIdx.x & 31;
    {
        const DaHead<D> t(p, b, kh * group);
        if (bad && (da_not_finite<D>(t.k + j * p.ld_kv) || da_not_finite<D>(t.v + j * p.ld_kv))) bad = false;
    }
    for (int h = kh * group; h < (kh + 1) * group; h++) {
        const DaHead<D> t(p, b, h);
        const uint32_t left = da_to_mend(bad, lo, hi, [&](int i) {
            return !(fabsf(t.lse[i]) < INFINITY) || !(fabsf(t.delta[i]) < INFINITY) || da_not_finite<D>(t.q + i * p.ld_q) || da_not_finite<D>(t.g + i * p.ld_out);
        });
        bad = left >> lane & 1;
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, bad); left; left &= left - 1) {
        const int r = __ffs(left) - 1, rj = __shfl_sync(0xffffffffu, j, r), from = __shfl_sync(0xffffffffu, lo, r), to = __shfl_sync(0xffffffffu, hi, r);
        float ak[D / 32] = {}, av[D / 32] = {};
        for (int h = kh * group; h < (kh + 1) * group; h++) {
            const DaHead<D> t(p, b, h);
            for (int i = from; i < to; i += 32) {
                float ds = 0.0f, w = 0.0f;
                if (i + lane < to) w = t.template pair<CAP>(p, i + lane, rj, ds);
                da_add_rows<D>(ak, ds, t.q + i * p.ld_q, p.ld_q, min(32, to - i));
                da_add_rows<D>(av, w, t.g + i * p.ld_out, p.ld_out, min(32, to - i));
            }
        }
        const int64_t at = ((int64_t)b * p.tokens + rj) * p.ld_dkv + kh * D;
        da_store_row<D>(p.dk + at, ak, p.scale);
        da_store_row<D>(p.dv + at, av, 1.0f);
    }
}

// ==========================================================================================================================
// forward
//
// An item is 256 queries of one head: two tiles of 128 that share the K and V tiles.  Each tile has its own score columns
// in tensor memory, its own output accumulator and its own eight softmax warps, two threads per query.  While one tile's
// warps exponentiate, the tensor core works for the other: S0 S1 | PV0 S0' | PV1 S1' | ...  Probabilities go back to
// tensor memory, over the scores they came from, as the A operand of P V: they never pass through shared memory, whose
// bandwidth the two operands of Q K^T already need.  A tile's next scores may be issued right behind its P V without a
// wait, since the tensor core works off its instructions in order.
// Keys are walked from the last block to the first: with the distance bias the largest scores come first, and the running
// maximum settles in the first block or two.  It is lazy besides: probabilities are taken relative to a reference that
// moves (and the accumulator is rescaled) only when the true maximum has run ahead of it by 2^8, so that P stays far inside fp16; fp16 and not fp32
// because it is the tensor core's operand type: 2^-11 of each probability, the same as V's own rounding.
//
// 8 rows of 2048, documents of 1200, 32 heads of 128, bias: 262 us.  8192 tokens in documents of 4500, 32 heads over 8, cap 50: 736 us, 456 TFLOP/s
// over visible pairs, the tensor pipe 30 % active.  A pair of tile steps takes 4400 to 5200 clocks: 2048 of the tensor core,
// and 3150 of the softmax warps, which wait for the scores of their own tile; a second score buffer per tile, which would
// take that wait away, has no room beside two accumulators of 128 columns in 512 columns of tensor memory.
// ==========================================================================================================================
template <int D>
struct FwdSmem {
    static constexpr uint32_t TILE = 128 * D * 2;
    static constexpr int SLOTS = 3;                     // of the ring that K and V tiles pass through in turn
    static constexpr size_t BYTES = 1024 + TILE * (2 + SLOTS) + 16 * DA_PATCH + sizeof(DaTable) + 256 + 2 * 4 * 2 * 128 * sizeof(float);
};

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DA_THREADS, 1)
doc_attn_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                    const __grid_constant__ CUtensorMap tmap_out,
                    const __grid_constant__ DocAttn p) {
    using S = FwdSmem<D>;
    constexpr uint32_t TMEM_COLS = 512;                 // S0 [0,128)  S1 [128,256)  O0 [256,256+D)  O1 [256+D,256+2D)
    constexpr uint32_t IDESC_S = make_idesc_f16_f32(128, 128, 0, 0);
    constexpr uint32_t IDESC_PV = make_idesc_f16_f32(128, D, 0, 1);
    constexpr float RESCALE_STEP = 8.0f;                // log2 units the row maximum may run ahead of the reference

    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = base;                           // two tiles
    unsigned char* sKV = sQ + 2 * S::TILE;              // the ring: K V K V ..
    unsigned char* sOut = sKV + S::SLOTS * S::TILE;     // a patch for each owner warp
    DaTable* table = reinterpret_cast<DaTable*>(sOut + 16 * DA_PATCH);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + 1);
    uint64_t* q_full = bars;                 // 2 (per tile)
    uint64_t* q_empty = bars + 2;            // 2
    uint64_t* kv_full = bars + 4;            // SLOTS
    uint64_t* kv_empty = bars + 8;           // SLOTS
    uint64_t* s_full = bars + 12;            // 2 (per tile)
    uint64_t* p_full = bars + 14;            // 2
    uint64_t* o_done = bars + 16;            // 2: a P V product of the tile is complete
    uint64_t* o_empty = bars + 18;           // 2: the tile's output has been read
    uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(bars + 20);
    float* exchange = reinterpret_cast<float*>(bars + 32);       // [tile][maxima of even, of odd blocks, sums, flags][owner][row]

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int per_row = (p.tokens + 255) / 256, n_tiles = p.batch * per_row;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::SLOTS; i++) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 8);
            mbar_init(&o_done[t], 1);
            mbar_init(&o_empty[t], 8);
        }
        fence_barrier_init();
        prefetch_tensormap(&tmap_q);
        prefetch_tensormap(&tmap_k);
        prefetch_tensormap(&tmap_v);
    }
    if (warp == 1) {
        tmem_alloc(tmem_base_smem, TMEM_COLS);
        tmem_relinquish();
    }
    pdl_wait();
    auto ranges = [&](int b, int t0, bool second) { return da_blocks<true>(p, b, second ? t0 + 128 : t0, 128); };
    const int listed = da_plan_items(table, n_tiles, p.heads, per_row, 256, ranges);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = uniform(*tmem_base_smem);
    const int group = p.heads / p.kv_heads;

    struct Item : DaItem {
        int last, n;         // the n blocks up to `last` that either tile needs, walked from the last one down
    };
    auto item_of = [&](int round, Item& m) {
        if (round < listed) static_cast<DaItem&>(m) = table->items[round];
        else if (listed < DA_LIST || !da_find_item(round, n_tiles, p.heads, per_row, 256, table, ranges, m)) return false;
        const bool has0 = m.r0.end > m.r0.begin, has1 = m.r1.end > m.r1.begin;
        m.last = max(m.r0.end, m.r1.end) - 1;
        m.n = m.last + 1 - (has0 ? (has1 ? min(m.r0.begin, m.r1.begin) : m.r0.begin) : m.r1.begin);
        return true;
    };

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            bool ok = true;
            uint32_t u = 0, q_count0 = 0, q_count1 = 0;         // loads through the ring: K of block n is 2n, V is 2n + 1
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                const int row = m.b * p.tokens, col = m.head * D, kcol = m.head / group * D;
                auto load_q = [&](int t, const Range& r, uint32_t& count) {
                    if (r.end == r.begin) return true;
                    if (!mbar_wait(&q_empty[t], (count++ & 1) ^ 1)) return false;       // the previous item's scores no longer read Q
                    mbar_arrive_expect_tx(&q_full[t], S::TILE);
#pragma unroll
                    for (int a = 0; a < D / 64; a++) tma_load_2d(sQ + t * S::TILE + a * 16384, &tmap_q, &q_full[t], col + a * 64, row + m.t0 + t * 128);
                    return true;
                };
                auto load = [&](const CUtensorMap* map, int y) {
                    const int s = u % S::SLOTS;
                    if (!mbar_wait(&kv_empty[s], ((u / S::SLOTS) & 1) ^ 1)) return false;
                    u++;
                    mbar_arrive_expect_tx(&kv_full[s], S::TILE);
#pragma unroll
                    for (int a = 0; a < D / 64; a++) tma_load_2d(sKV + s * S::TILE + a * 16384, map, &kv_full[s], kcol + a * 64, y);
                    return true;
                };
                // the second tile begins first, where its keys reach further
                const bool second = m.r1.end > m.r0.end;
                if (second) ok = load_q(1, m.r1, q_count1) && load_q(0, m.r0, q_count0);
                else ok = load_q(0, m.r0, q_count0) && load_q(1, m.r1, q_count1);
                for (int n = 0; n < m.n && ok; n++) ok = load(&tmap_k, row + (m.last - n) * 128) && load(&tmap_v, row + (m.last - n) * 128);
            }
            if (!ok) atomicExch(&g_doc_error, 1);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: the warp walks and waits together, which keeps addresses and descriptors in uniform
        // registers; one lane issues ----------------
        {
            const bool issuer = elect_one();
            bool ok = true;
            uint32_t it = 0, q_count0 = 0, q_count1 = 0, p_count0 = 0, p_count1 = 0;        // blocks, and per tile: items, blocks
            const uint64_t q_desc = make_smem_desc_sw128(smem_u32(sQ), 16, 1024), k_desc = make_smem_desc_sw128(smem_u32(sKV), 16, 1024);
            const uint64_t v_desc = make_smem_desc_sw128(smem_u32(sKV), 16384, 1024);
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                m.last = uniform(m.last), m.n = uniform(m.n);
                m.r0.begin = uniform(m.r0.begin), m.r0.end = uniform(m.r0.end), m.r1.begin = uniform(m.r1.begin), m.r1.end = uniform(m.r1.end);
                for (int n = -1; n < m.n && ok; n++) {
                    const uint32_t v_load = 2 * (it + n) + 1, k_load = v_load + 1;               // n == -1 uses no V
                    const int vs = v_load % S::SLOTS, ks = k_load % S::SLOTS;
                    const bool more = n + 1 < m.n;
                    const int blk = m.last - n;
                    if (n >= 0) ok = mbar_wait(&kv_full[vs], (v_load / S::SLOTS) & 1);
                    if (ok && more) ok = mbar_wait(&kv_full[ks], (k_load / S::SLOTS) & 1);
                    // P V of block n and then the scores of block n + 1; the index is a constant, so that nothing lands in local memory
                    auto step = [&](auto tile, const Range& r, uint32_t& q_count, uint32_t& p_count) {
                        constexpr int t = decltype(tile)::value;
                        if (n >= 0 && blk >= r.begin && blk < r.end) {
                            const bool first = blk == r.end - 1;
                            if (!mbar_wait(&p_full[t], p_count & 1)) return false;
                            if (first && !mbar_wait(&o_empty[t], q_count & 1)) return false;       // the count is one ahead: this item's scores are out
                            tcgen05_fence_after();
                            const uint64_t vd = v_desc + (uint32_t)(vs * (S::TILE >> 4));
                            if (issuer) {
#pragma unroll
                                for (int kk = 0; kk < 8; kk++)        // A = P [128 q x 128 keys] in tensor memory, B = V [128 keys x D], d contiguous
                                    umma_f16_ts(tmem_base + 256 + t * D, tmem_base + t * 128 + (kk >> 2) * 64 + (kk & 3) * 8, vd + kk * 128, IDESC_PV, kk != 0 || !first ? 1u : 0u);
                                umma_commit(&o_done[t]);
                            }
                            p_count++;
                        }
                        if (more && blk - 1 >= r.begin && blk - 1 < r.end) {
                            if (blk == r.end && !mbar_wait(&q_full[t], q_count++ & 1)) return false;
                            tcgen05_fence_after();
                            const uint64_t qd = q_desc + t * (S::TILE >> 4), kd = k_desc + (uint32_t)(ks * (S::TILE >> 4));
                            if (issuer) {
#pragma unroll
                                for (int kk = 0; kk < D / 16; kk++) {
                                    const int off = (kk >> 2) * 1024 + (kk & 3) * 2;
                                    umma_f16_ss(tmem_base + t * 128, qd + off, kd + off, IDESC_S, kk != 0 ? 1u : 0u);
                                }
                                umma_commit(&s_full[t]);
                                if (blk - 1 == r.begin) umma_commit(&q_empty[t]);
                            }
                        }
                        return true;
                    };
                    ok = ok && step(std::integral_constant<int, 0>(), m.r0, q_count0, p_count0) && step(std::integral_constant<int, 1>(), m.r1, q_count1, p_count1);
                    if (!ok) break;
                    if (issuer) {
                        if (n >= 0) umma_commit(&kv_empty[vs]);
                        if (more) umma_commit(&kv_empty[ks]);
                    }
                }
                it += m.n;
            }
            if (!ok && issuer) atomicExch(&g_doc_error, 2);
        }
    } else {
        // ---------------- softmax / epilogue: two threads per query, 64 of the 128 key columns each ----------------
        const int t = (warp - 2) >> 3, half = (warp - 2) >> 2 & 1;
        const int quarter = warp & 3;                   // a warp reaches tensor-memory lanes 32 * (warp % 4) ..
        const int r = quarter * 32 + lane;
        const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tm_s = tm + t * 128 + half * 64, tm_o = tm + 256 + t * D + half * (D / 2);
        float* const cells = exchange + t * 1024 + r;
        unsigned char* const patch = sOut + (warp - 2) * DA_PATCH;
        // The owners of 32 rows meet once a block.  Every owner reaches it in every block, also one whose bounded wait gave up.
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + quarter) : "memory"); };
        bool ok = true;
        uint32_t it = 0;
        Item m = {};
        auto span_of = [&]() {
            const int qi = m.t0 + t * 128 + r;
            // rows behind the sequence never force the masked path
            return qi < p.tokens ? p.spans[(int64_t)m.b * p.tokens + qi] : make_int4(0, 0x7fffffff, 0, 0);
        };
        bool have = item_of(0, m);
        int4 span = make_int4(0, 0, 0, 0);
        float slope = 0.0f;
        if (have) {
            span = span_of();
            if (BIAS) slope = p.slopes[m.head];
        }
        for (int round = 1; have; round++) {
            const Range blocks = t == 0 ? m.r0 : m.r1;
            const int head = m.head, b = m.b, qi = m.t0 + t * 128 + r;
            const bool live = qi < p.tokens;
            const int64_t row = (int64_t)b * p.tokens + qi;
            const int lo = max(span.x, 0), hi = live ? min(span.y, p.tokens) : span.y;
            const float slope2 = slope * LOG2E;
            have = item_of(round, m);                   // the next item's span and slope travel while this one is worked on
            if (have) {
                span = span_of();
                if (BIAS) slope = p.slopes[m.head];
            }
            float* lse = p.lse && half == 0 ? p.lse + ((int64_t)b * p.heads + head) * p.tokens + qi : nullptr;
            if (blocks.end == blocks.begin) {
                if (live) {
                    da_zero_row(p.out + row * p.ld_out + head * D + half * (D / 2), D / 2);
                    if (lse) *lse = 0.0f;
                }
                continue;
            }
            const bool ahead = BIAS && __any_sync(0xffffffffu, live && hi > qi + 1);      // some row sees keys behind itself: the prompt's
            float m_ref = -INFINITY;
            float2 l = both(0.0f);
            for (int blk = blocks.end - 1; blk >= blocks.begin; blk--, it++) {
                if (ok) ok = mbar_wait(&s_full[t], it & 1);
                ok = __all_sync(0xffffffffu, ok);
                // The scores are read twice, 32 columns at a time: once for the maximum, once for the exponentials.  Keeping all of
                // a row's in registers instead made straight-line code of some 1400 instructions a block, which the warps could
                // not run through in less than 5 clocks each.
                const int kbase = blk * 128 + half * 64;
                uint32_t part = 0, whole = 0;                         // which chunks some row of the warp sees, and all rows see throughout
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int k0 = kbase + c * 32;
                    if (lo < k0 + 32 && hi > k0) part |= 1u << c;
                    if (lo <= k0 && hi >= k0 + 32 && (!BIAS || !ahead || k0 + 31 <= qi)) whole |= 1u << c;
                }
                part = __reduce_or_sync(0xffffffffu, part);
                whole = __reduce_and_sync(0xffffffffu, whole);
                const float dist = (float)(kbase - qi), slant = slope2 * dist;
                bool near = true;                       // the polynomial reaches every argument of the cap's tanh in this warp's part of the block
                // Chunk c of the scores plus `shift`, in log2 units; what is masked is -inf.  RAW: as the products are, which is enough for
                // the maximum where there is no bias (the scale and the cap keep the order).
                auto scores = [&](int c, float2(&x)[16], float shift, auto raw) {
                    constexpr bool RAW = decltype(raw)::value;
                    tmem_ld_32x32b_x32(tm_s + c * 32, reinterpret_cast<float*>(x));
                    tmem_ld_wait();
                    if (CAP && (RAW || BIAS)) {
                        float wide = 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; i++) wide = max3(wide, fabsf(x[i].x), fabsf(x[i].y));
                        near = __all_sync(0xffffffffu, wide * p.cap_in <= TANH_REACH) && near;
                    }
                    auto fill = [&](auto line) {        // line: the bias as a straight line in the key's number
                        constexpr bool LINE = BIAS && decltype(line)::value;
                        const float2 at = both(shift);
                        Line bias(LINE ? slope2 : 0.0f, LINE ? fmaf(slope2, (float)(c * 32), slant) + shift : 0.0f);
                        if (CAP && near) {
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = da_capped_near(x[i], p, LINE ? bias.next(i) : at);
                        } else if (CAP) {
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = __fadd2_rn(da_capped_far(x[i], p), LINE ? bias.next(i) : at);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = __ffma2_rn(x[i], both(p.scale_log2), LINE ? bias.next(i) : at);
                        }
                    };
                    if (whole >> c & 1) {
                        if (!RAW) fill(Flag<true>());
                    } else {
                        if (!RAW) fill(Flag<false>());
                        const float d0 = dist + (float)(c * 32);
                        const uint32_t seen = span_bits(lo - kbase - c * 32, hi - kbase - c * 32);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            if (BIAS && !RAW) {
                                x[i].x = fmaf(-slope2, fabsf(d0 + (float)(2 * i)), x[i].x);
                                x[i].y = fmaf(-slope2, fabsf(d0 + (float)(2 * i + 1)), x[i].y);
                            }
                            x[i].x = seen & 1u << (2 * i) ? x[i].x : -INFINITY;
                            x[i].y = seen & 2u << (2 * i) ? x[i].y : -INFINITY;
                        }
                    }
                };
                float top = -INFINITY;
                if (ok) {
                    tcgen05_fence_after();
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
                        if (!(part >> c & 1)) continue;
                        float2 x[16];
                        scores(c, x, 0.0f, Flag<!BIAS>());
                        float t4[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 16; i++) t4[i & 3] = max3(t4[i & 3], x[i].x, x[i].y);
                        top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                    }
                }
                float* const cell = cells + (it & 1) * 256;           // two turns, so that one meeting a block is enough
                cell[half * 128] = top;
                meet();
                top = fmaxf(top, cell[(half ^ 1) * 128]);
                if (!ok) continue;
                if (CAP && !BIAS) top = top == -INFINITY ? top : da_tanh(top * p.cap_in) * p.cap_log2;
                if (!CAP && !BIAS) top *= p.scale_log2;
                const bool move = top > m_ref + RESCALE_STEP;        // also the row's first visible key (m_ref = -inf)
                float factor = 1.0f;
                if (move) {
                    factor = m_ref == -INFINITY ? 0.0f : fast_exp2(m_ref - top);
                    m_ref = top;
                    l = __fmul2_rn(l, both(factor));
                }
                if (blk < blocks.end - 1 && __any_sync(0xffffffffu, move)) {
                    // the accumulator may only be touched between two P V products: wait for the previous one
                    ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (it - 1) & 1));
                    if (!ok) continue;
                    tcgen05_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 32) {
                        uint32_t v[32];
                        tmem_ld_32x32b_x32(tm_o + c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * factor);
                        tmem_st_32x32b_x32(tm_o + c, v);
                    }
                }
                const float shift = m_ref == -INFINITY ? 0.0f : -m_ref;        // nothing visible yet: every exponential is 0
#pragma unroll 1
                for (int c = 0; c < 2; c++) {
                    uint32_t w[16];
                    if (part >> c & 1) {
                        float2 x[16];
                        scores(c, x, shift, Flag<false>());
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float2 pe = make_float2(fast_exp2(x[i].x), fast_exp2(x[i].y));
                            l = __fadd2_rn(l, pe);
                            w[i] = da_half2(pe.x, pe.y);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++) w[i] = 0;
                    }
                    tmem_st_32x32b_x16(tm_s + c * 16, w);             // over this owner's scores that have been read: columns below 32 (c + 1)
                }
                tmem_st_wait();
                tcgen05_fence_before();
                warp_arrive(&p_full[t]);
            }
            // epilogue: O / l -> fp16, token-major; log-sum-exp for the backward
            float* const sums = cells + 512;
            sums[half * 128] = l.x + l.y;
            meet();
            const float sum = sums[0] + sums[128];
            if (ok) ok = mbar_wait(&o_done[t], (it - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);        // a NaN stays one
            const float lse2 = m_ref + __log2f(sum);
            const bool none = lo >= hi;
            __half2 bad[2] = {__float2half2_rn(0.0f), __float2half2_rn(0.0f)};
            if (ok) {
                tcgen05_fence_after();
#pragma unroll
                for (int c = 0; c < D / 2; c += 32) {
                    float2 x[16];
                    tmem_ld_32x32b_x32(tm_o + c, reinterpret_cast<float*>(x));
                    tmem_ld_wait();
                    if (c + 32 == D / 2) {
                        tcgen05_fence_before();
                        warp_arrive(&o_empty[t]);
                    }
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 y = __fmul2_rn(x[i], both(inv));
                        w[i] = da_half2(y.x, y.y);
                        bad[i & 1] = __hfma2(*reinterpret_cast<const __half2*>(&w[i]), __float2half2_rn(0.0f), bad[i & 1]);      // a NaN, once something is not finite
                        if (none) w[i] = 0;
                    }
                    da_patch_free();
#pragma unroll
                    for (int i = 0; i < 4; i++) da_stage<32>(patch, lane, i, w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    da_patch_store(&tmap_out, patch, head * D + half * (D / 2) + c, qi - lane, b, p.tokens);
                }
                if (live && lse) *lse = none ? 0.0f : lse2 * LN2;
            }
            const __half2 any = __hadd2(bad[0], bad[1]);
            const bool again = ok && live && !none && fabsf(lse2) < INFINITY && (__hisnan(__low2half(any)) || __hisnan(__high2half(any)));
            if (barrier_any(1 + t * 4 + quarter, 64, again)) {
                float* const flags = cells + 768;
                flags[half * 128] = again ? 1.0f : 0.0f;
                da_patch_written();
                meet();                                 // orders both owners' stores before a row is written again
                const bool redo = flags[0] + flags[128] != 0.0f;
                if (half == 0) da_mend_out<D, CAP>(p, b, head, qi, lo, hi, lse2, redo);
                meet();
            }
        }
        da_patch_free();                                // the patch is read before the CTA's shared memory goes
        if (!ok && lane == 0) atomicExch(&g_doc_error, 3);
    }

    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// ==========================================================================================================================
// backward
//
// delta first, then two kernels that each form the probabilities again from the saved log-sum-exp: one owns 128 keys and
// walks the queries that see them (dK, dV), one owns 128 queries and walks their keys (dQ).  Seven products instead of
// the five of a single kernel, but no atomic additions into dQ, whose order would change the result from run to run.
// Four threads share a row (warps w, w + 4, w + 8 and w + 12 own the same 32 tensor-memory lanes and split the columns):
// with two, a scheduler had too few warps to hide the latency of their own loads and exponentials.  P and dS return to tensor
// memory over the scores they came from, as A operands; each quarter of the columns stays inside its own quarter of the
// region, so no owner overwrites what another has yet to read.  They are rounded to fp16 there, as operands have to be.
//
// 2 rows of 1024 tokens, documents of 300, 32 heads of 128: 79 us for the three; 8192 tokens, documents of
// 4500, 32 heads over 8, cap 50: 1826 us, 643 TFLOP/s of the seven products over visible pairs, the tensor pipe 39 %
// (dK, dV) and 49 % (dQ) of the time active.  What bounds them is the owners' issue slots: cap, exponential and derivative
// are about 25 instructions a pair of scores.
// delta comes from O as the forward rounded it, which adds up to 1.6e-4 of dQ and dK where documents are long (dS as an fp16
// operand adds 2.0e-4, their own rounding 2.1e-4) and 6e-4 in documents of two tokens, where dP and delta nearly cancel; the
// exact sum of P dP would take two more products before the first dS.
// ==========================================================================================================================

// delta_i = sum_d dO_id O_id per query and head: a CTA per token, d / 8 neighbouring lanes own one head
__global__ void __launch_bounds__(256)
doc_delta_kernel(const __half* out, const __half* dout, int64_t ld, float* delta, int tokens, int heads, int d) {
    const int lanes = d >> 3, pieces = heads * lanes, row = blockIdx.x;
    const int b = row / tokens;
    float* const to = delta + (int64_t)b * heads * tokens + (row - b * tokens);
    pdl_wait();
    pdl_launch_dependents();
    const __half* o = out + row * ld;
    const __half* g = dout + row * ld;
    for (int i0 = 0; i0 < pieces; i0 += 256) {
        const int i = i0 + threadIdx.x;
        float2 s = make_float2(0.0f, 0.0f);
        if (i < pieces) {
            const uint4 a = ld_raw(o + i * 8), c = ld_raw(g + i * 8);
            const __half2 *x = reinterpret_cast<const __half2*>(&a), *y = reinterpret_cast<const __half2*>(&c);
#pragma unroll
            for (int e = 0; e < 4; e++) s = __ffma2_rn(__half22float2(x[e]), __half22float2(y[e]), s);
        }
        float sum = s.x + s.y;
        for (int w = lanes >> 1; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (i < pieces && (i & (lanes - 1)) == 0) to[(int64_t)(i / lanes) * tokens] = sum;
    }
}

constexpr int DA_SUB = 64;                  // queries per step of the dK / dV kernel
constexpr uint32_t DA_SUB_ATOM = DA_SUB * 128;

template <int D>
struct DkvSmem {
    static constexpr uint32_t KV = 128 * D * 2, SUB = DA_SUB * D * 2;
    static constexpr int STAGES = 3;
    static constexpr size_t BYTES = 1024 + 2 * KV + 2 * STAGES * SUB + 16 * DA_PATCH + 4 * 2 * DA_SUB * sizeof(float) + sizeof(DaTable) + 256;
};

// Transposed scores S^T = K Q^T and dP^T = V dO^T (a row owner is a key), so that P^T and dS^T are the A operands of
// dV += P^T dO and dK += dS^T Q as they stand; the 64 queries' lse and delta of a step come from shared memory.  With
// shared key heads the walk goes over all query heads of the group, and the sum over them stays in the accumulators.
template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DA_THREADS, 1)
doc_attn_dkv_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                    const __grid_constant__ CUtensorMap tmap_do, const __grid_constant__ CUtensorMap tmap_dk, const __grid_constant__ CUtensorMap tmap_dv,
                    const __grid_constant__ DocAttn p) {
    using S = DkvSmem<D>;
    constexpr uint32_t TMEM_COLS = 512;     // S^T x2 [0,128)  dP^T x2 [128,256)  dV [256,256+D)  dK [256+D,256+2D)
    constexpr uint32_t IDESC_ST = make_idesc_f16_f32(128, DA_SUB, 0, 0);
    constexpr uint32_t IDESC_ACC = make_idesc_f16_f32(128, D, 0, 1);

    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sK = base;
    unsigned char* sV = sK + S::KV;
    unsigned char* sQ = sV + S::KV;
    unsigned char* sDO = sQ + S::STAGES * S::SUB;
    unsigned char* sOut = sDO + S::STAGES * S::SUB;     // a patch for each owner warp
    float* stat = reinterpret_cast<float*>(sOut + 16 * DA_PATCH);       // [team][2][lse2 x 64 | delta x 64]
    DaTable* table = reinterpret_cast<DaTable*>(stat + 4 * 2 * DA_SUB);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + 1);
    uint64_t* kv_full = bars;
    uint64_t* kv_empty = bars + 1;
    uint64_t* q_full = bars + 2;       // STAGES
    uint64_t* q_empty = bars + 6;      // STAGES
    uint64_t* s_full = bars + 10;      // 2
    uint64_t* p_full = bars + 12;      // 2
    uint64_t* acc_full = bars + 14;
    uint64_t* acc_empty = bars + 15;
    uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(bars + 16);

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int per_row = (p.tokens + 127) / 128, n_tiles = p.batch * per_row;
    const int group = p.heads / p.kv_heads;

    if (threadIdx.x == 0) {
        mbar_init(kv_full, 1);
        mbar_init(kv_empty, 1);
        for (int i = 0; i < S::STAGES; i++) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 8);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_base_smem, TMEM_COLS);
        tmem_relinquish();
    }
    auto ranges = [&](int b, int t0, bool second) { return second ? Range{0, 0} : da_blocks<false>(p, b, t0, DA_SUB); };
    const int listed = da_plan_items(table, n_tiles, p.kv_heads, per_row, 128, ranges);
    // Everything before the delta kernel is complete when this one starts: only delta is waited for.  The dQ kernel needs nothing of
    // this one and may take over each SM that is done here.
    pdl_wait();
    pdl_launch_dependents();
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = uniform(*tmem_base_smem);

    struct Item : DaItem {
        int n;                 // steps: 64-query blocks r0, times query heads of the group
    };
    auto item_of = [&](int round, Item& m) {
        if (round < listed) static_cast<DaItem&>(m) = table->items[round];
        else if (listed < DA_LIST || !da_find_item(round, n_tiles, p.kv_heads, per_row, 128, table, ranges, m)) return false;
        m.n = (m.r0.end - m.r0.begin) * group;
        return true;
    };

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            uint32_t it = 0, items = 0;
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                if (m.n == 0) continue;
                const int row = m.b * p.tokens, kcol = m.head * D;
                ok = mbar_wait(kv_empty, (items++ & 1) ^ 1);       // the previous item's score products no longer read K / V
                if (!ok) break;
                mbar_arrive_expect_tx(kv_full, 2 * S::KV);
#pragma unroll
                for (int a = 0; a < D / 64; a++) {
                    tma_load_2d(sK + a * 16384, &tmap_k, kv_full, kcol + a * 64, row + m.t0);
                    tma_load_2d(sV + a * 16384, &tmap_v, kv_full, kcol + a * 64, row + m.t0);
                }
                int blk = m.r0.begin, col = m.head * group * D;
                for (int n = 0; n < m.n && ok; n++, it++) {
                    const int s = it % S::STAGES;
                    ok = mbar_wait(&q_empty[s], ((it / S::STAGES) & 1) ^ 1);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&q_full[s], 2 * S::SUB);
#pragma unroll
                    for (int a = 0; a < D / 64; a++) {
                        tma_load_2d(sQ + s * S::SUB + a * DA_SUB_ATOM, &tmap_q, &q_full[s], col + a * 64, row + blk * DA_SUB);
                        tma_load_2d(sDO + s * S::SUB + a * DA_SUB_ATOM, &tmap_do, &q_full[s], col + a * 64, row + blk * DA_SUB);
                    }
                    if (++blk == m.r0.end) {
                        blk = m.r0.begin;
                        col += D;
                    }
                }
            }
            if (!ok) atomicExch(&g_doc_error, 11);
        }
    } else if (warp == 1) {
        {
            bool ok = true;
            const bool issuer = elect_one();
            const uint64_t k_desc = make_smem_desc_sw128(smem_u32(sK), 16, 1024), v_desc = make_smem_desc_sw128(smem_u32(sV), 16, 1024);
            const uint64_t q_desc = make_smem_desc_sw128(smem_u32(sQ), 16, 1024), do_desc = make_smem_desc_sw128(smem_u32(sDO), 16, 1024);
            const uint64_t q_col = make_smem_desc_sw128(smem_u32(sQ), DA_SUB_ATOM, 1024), do_col = make_smem_desc_sw128(smem_u32(sDO), DA_SUB_ATOM, 1024);
            uint32_t it0 = 0, items = 0;
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                m.n = uniform(m.n);
                if (m.n == 0) continue;
                ok = mbar_wait(kv_full, items & 1);
                // step n issues the transposed scores of block n and then the accumulations of block n - 1, whose P^T / dS^T
                // the row owners produced meanwhile; buffer n & 1 was last read by the accumulations of n - 2, issued before
                for (int n = 0; n <= m.n && ok; n++) {
                    if (n < m.n) {
                        const uint32_t i = it0 + n;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&q_full[s], (i / S::STAGES) & 1);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint64_t qd = q_desc + (uint32_t)(s * (S::SUB >> 4)), dod = do_desc + (uint32_t)(s * (S::SUB >> 4));
                        if (issuer) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; kk++)      // S^T = K Q^T : [128 keys x 64 queries]
                                umma_f16_ss(tmem_base + sb * DA_SUB, k_desc + (kk >> 2) * 1024 + (kk & 3) * 2, qd + (kk >> 2) * (DA_SUB_ATOM >> 4) + (kk & 3) * 2,
                                            IDESC_ST, kk != 0 ? 1u : 0u);
#pragma unroll
                            for (int kk = 0; kk < D / 16; kk++)      // dP^T = V dO^T
                                umma_f16_ss(tmem_base + 128 + sb * DA_SUB, v_desc + (kk >> 2) * 1024 + (kk & 3) * 2, dod + (kk >> 2) * (DA_SUB_ATOM >> 4) + (kk & 3) * 2,
                                            IDESC_ST, kk != 0 ? 1u : 0u);
                            umma_commit(&s_full[sb]);
                            if (n == m.n - 1) umma_commit(kv_empty);       // last products of the item that read K / V
                        }
                    }
                    if (n >= 1) {
                        const uint32_t i = it0 + n - 1;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&p_full[sb], (i >> 1) & 1);
                        if (ok && n == 1) ok = mbar_wait(acc_empty, (items & 1) ^ 1);      // the previous item's dV / dK have been read
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint64_t qd = q_col + (uint32_t)(s * (S::SUB >> 4)), dod = do_col + (uint32_t)(s * (S::SUB >> 4));
                        if (issuer) {
#pragma unroll
                            for (int kk = 0; kk < DA_SUB / 16; kk++)      // dV += P^T dO (contraction over the 64 queries)
                                umma_f16_ts(tmem_base + 256, tmem_base + sb * DA_SUB + kk * 16, dod + kk * 128, IDESC_ACC,
                                            n != 1 || kk != 0 ? 1u : 0u);
#pragma unroll
                            for (int kk = 0; kk < DA_SUB / 16; kk++)      // dK += dS^T Q
                                umma_f16_ts(tmem_base + 256 + D, tmem_base + 128 + sb * DA_SUB + kk * 16, qd + kk * 128, IDESC_ACC,
                                            n != 1 || kk != 0 ? 1u : 0u);
                            umma_commit(&q_empty[s]);
                        }
                    }
                }
                if (ok && issuer) umma_commit(acc_full);
                it0 += m.n;
                items++;
            }
            if (!ok && issuer) atomicExch(&g_doc_error, 12);
        }
    } else {
        // ---------------- row owners ----------------
        // Two groups of eight warps take the steps in turn, each with a score buffer of its own, so that one loads and stores
        // while the other computes; in a group two threads share a key, 32 of the 64 query columns each.  The results are shared
        // by all: a quarter of the columns each.
        const int quarter = warp & 3, part = (warp - 2) >> 2, team = part >> 1, half = part & 1;
        const int r = quarter * 32 + lane;
        const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16);
        unsigned char* const patch = sOut + (warp - 2) * DA_PATCH;
        bool ok = true;
        uint32_t it0 = 0, items = 0;
        Item m = {}, following = {};
        int4 next_span = make_int4(0, 0, 0, 0);
        float next = 0.0f, next_slope = 0.0f;
        // A step's 64 log-sum-exps and 64 deltas, one for each of the team's first owners, fetched a step ahead as they are:
        // arithmetic on them would wait for the load where it is issued.  Step n of an item; the blocks repeat for every head.
        auto fetch = [&](const Item& of, int blk, int h) {
            const int i = blk * DA_SUB + (r & 63);
            next = 0.0f;
            if (half == 0 && i < p.tokens) next = (r < 64 ? p.lse_in : p.delta)[((int64_t)of.b * p.heads + h) * p.tokens + i];
            if (BIAS) next_slope = p.slopes[h];
        };
        // the team's first step of an item whose steps are counted from `from`
        auto fetch_first = [&](const Item& of, uint32_t from) {
            const int n = (from & 1) != (uint32_t)team, wide = of.r0.end - of.r0.begin;
            if (n < of.n) fetch(of, of.r0.begin + (wide > 1 ? n : 0), of.head * group + (wide > 1 ? 0 : n));
        };
        auto team_meet = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(1 + team) : "memory"); };
        auto fetch_span = [&]() {
            const int kj = following.t0 + r;
            // rows behind the sequence never force the masked path
            next_span = kj < p.tokens ? p.spans[(int64_t)following.b * p.tokens + kj] : make_int4(0, 0, 0, 0x7fffffff);
        };
        bool have = item_of(0, following);
        if (have) {
            fetch_span();
            fetch_first(following, 0);
        }
        for (int round = 1; have; round++) {
            m = following;
            const int4 span = next_span;
            have = item_of(round, following);           // the next item's span and first statistics travel while this one is worked on
            if (have) fetch_span();
            const int kj = m.t0 + r;
            const bool live = kj < p.tokens;
            const int64_t row = (int64_t)m.b * p.tokens + kj;
            if (m.n == 0) {
                if (live) {
                    da_zero_row(p.dk + row * p.ld_dkv + m.head * D + part * (D / 4), D / 4);
                    da_zero_row(p.dv + row * p.ld_dkv + m.head * D + part * (D / 4), D / 4);
                }
                if (have) fetch_first(following, it0);
                continue;
            }
            const int qlo = max(span.z, 0), qhi = live ? min(span.w, p.tokens) : span.w;
            int blk = m.r0.begin, h = m.head * group;
            auto advance = [&]() {
                if (++blk == m.r0.end) {
                    blk = m.r0.begin;
                    h++;
                }
            };
            const int first = (it0 & 1) != (uint32_t)team;
            if (first) advance();
            if (first >= m.n && have) fetch_first(following, it0 + m.n);
            for (int n = first; n < m.n; n += 2) {
                const uint32_t i = it0 + n;
                const int sb = team, q0 = blk * DA_SUB;
                float* const own = stat + (sb * 2 + ((i >> 1) & 1)) * 128;
                const float slope2 = next_slope * LOG2E;
                // negated, and the log-sum-exp in log2 units with the query's share of the bias
                if (half == 0) own[r] = r < 64 ? fmaf(next, -LOG2E, -slope2 * (float)r) : -next;
                advance();
                advance();
                if (n + 2 < m.n) fetch(m, blk, h);
                else if (have) fetch_first(following, it0 + m.n);
                // orders this step's writes after the team's reads two steps of its own ago; every owner of the team reaches it in
                // every step, also one whose bounded wait gave up (it only skips the work)
                team_meet();
                if (ok) ok = mbar_wait(&s_full[sb], (i >> 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) continue;
                tcgen05_fence_after();
#pragma unroll 1
                for (int c0 = half * 32; c0 < half * 32 + 32; c0 += 16) {
                    const float4* nlse = reinterpret_cast<const float4*>(own + c0);
                    const float4* ndelta = nlse + 16;
                    float2 x[8], g[8];
                    tmem_ld_32x32b_x16(tm + sb * DA_SUB + c0, reinterpret_cast<float*>(x));
                    tmem_ld_32x32b_x16(tm + 128 + sb * DA_SUB + c0, reinterpret_cast<float*>(g));
                    tmem_ld_wait();
                    const float2 bias = both(slope2 * (float)(kj - q0));       // minus slope * (query - q0), which nlse holds
                    const bool inner = qlo <= q0 + c0 && qhi >= q0 + c0 + 16 && (!BIAS || kj <= q0 + c0);
                    const bool plain = __all_sync(0xffffffffu, inner);
                    bool near = true;
                    if (CAP) {
                        float wide = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; e++) wide = max3(wide, fabsf(x[e].x), fabsf(x[e].y));
                        near = __all_sync(0xffffffffu, wide * p.cap_in <= TANH_REACH);
                    }
                    auto step = [&](auto edge, auto reach) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float4 l4 = nlse[e >> 1], d4 = ndelta[e >> 1];
                            float2 off = e & 1 ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y);
                            const float2 nd = e & 1 ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);
                            if (BIAS) off = __fadd2_rn(off, bias);
                            const int far = q0 + c0 + 2 * e - kj;              // query - key
                            if (BIAS && edge) {                                // a key ahead of the query: -slope (key - query)
                                off.x += fminf(0.0f, 2.0f * slope2 * (float)far);
                                off.y += fminf(0.0f, 2.0f * slope2 * (float)(far + 1));
                            }
                            float2 s, t;
                            if (CAP) {
                                t = reach ? da_capped_near(x[e], p, both(0.0f)) : da_capped_far(x[e], p);
                                s = __fadd2_rn(t, off);
                            } else {
                                s = __ffma2_rn(x[e], both(p.scale_log2), off);
                            }
                            float2 pe = make_float2(fast_exp2(s.x), fast_exp2(s.y));
                            float2 de = __fmul2_rn(pe, __fadd2_rn(g[e], nd));
                            if (CAP) de = __fmul2_rn(de, __ffma2_rn(__fmul2_rn(t, both(p.cap_curve)), t, both(1.0f)));
                            if (edge) {
                                const int qi = q0 + c0 + 2 * e;
                                if (!(qlo <= qi && qi < qhi)) pe.x = de.x = 0.0f;
                                if (!(qlo <= qi + 1 && qi + 1 < qhi)) pe.y = de.y = 0.0f;
                            }
                            x[e].x = __uint_as_float(da_half2(pe.x, pe.y));
                            g[e].x = __uint_as_float(da_half2(de.x, de.y));
                        }
                    };
                    if (near) {
                        if (plain) step(Flag<false>(), Flag<true>());
                        else step(Flag<true>(), Flag<true>());
                    } else {
                        step(Flag<true>(), Flag<false>());
                    }
                    uint32_t wp[8], wd[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        wp[e] = __float_as_uint(x[e].x);
                        wd[e] = __float_as_uint(g[e].x);
                    }
                    tmem_st_32x32b_x8(tm + sb * DA_SUB + c0, wp);
                    tmem_st_32x32b_x8(tm + 128 + sb * DA_SUB + c0, wd);
                }
                tmem_st_wait();
                tcgen05_fence_before();
                warp_arrive(&p_full[sb]);
            }
            it0 += m.n;
            if (ok) ok = mbar_wait(acc_full, items & 1);
            ok = __all_sync(0xffffffffu, ok);
            items++;
            float bad = 0.0f;
            const bool none = qlo >= qhi;
            if (ok) {
                tcgen05_fence_after();
#pragma unroll
                for (int k = 0; k < 2; k++) {              // dV, then dK: D / 4 columns of each
                    uint32_t w[D / 8];
#pragma unroll
                    for (int c = 0; c < D / 4; c += 16) {
                        float2 a[8];
                        tmem_ld_32x32b_x16(tm + 256 + k * D + part * (D / 4) + c, reinterpret_cast<float*>(a));
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            bad = fmaf(a[i].x, 0.0f, fmaf(a[i].y, 0.0f, bad));
                            w[c / 2 + i] = none ? 0 : k == 0 ? da_half2(a[i].x, a[i].y) : da_half2(a[i].x * p.scale, a[i].y * p.scale);
                        }
                    }
                    if (k == 1) {
                        tcgen05_fence_before();
                        warp_arrive(acc_empty);            // the accumulators may take the next item's first products
                    }
                    da_patch_free();
#pragma unroll
                    for (int i = 0; i < D / 32; i++) da_stage<D / 4>(patch, lane, i, w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    da_patch_store(k == 0 ? &tmap_dv : &tmap_dk, patch, m.head * D + part * (D / 4), kj - lane, m.b, p.tokens);
                }
            }
            // evaluated again by the warps of the rows' first owners, after all owners' stores
            const bool again = ok && live && !none && bad != 0.0f;
            if (barrier_any(3, 512, again)) {
                if (part == 0) stat[r] = 0.0f;
                asm volatile("bar.sync 3, 512;" ::: "memory");
                if (again) stat[r] = 1.0f;
                da_patch_written();
                asm volatile("bar.sync 3, 512;" ::: "memory");
                const bool redo = stat[r] != 0.0f;
                if (part == 0 && __any_sync(0xffffffffu, redo)) da_mend_dkv<D, CAP>(p, m.b, m.head, kj, qlo, qhi, redo);
                asm volatile("bar.sync 3, 512;" ::: "memory");
            }
        }
        da_patch_free();                                // the patch is read before the CTA's shared memory goes
        if (!ok && lane == 0) atomicExch(&g_doc_error, 13);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

template <int D>
struct DqSmem {
    static constexpr uint32_t TILE = 128 * D * 2;
    static constexpr int STAGES = 2;
    static constexpr int PATCH = DA_PATCH / 2;          // 16 columns at a time: Q, dO and two stages of K and V leave no more
    static constexpr size_t BYTES = 1024 + 2 * TILE + 2 * STAGES * TILE + 16 * PATCH + 128 * sizeof(float) + sizeof(DaTable) + 256;
};

// S = Q K^T (two buffers), dP = dO V^T (one), dQ += dS K over blocks of 128 keys.  dS goes over the scores it came from,
// so dP's buffer is free as soon as the owners have read it: S(n+1) and dP(n+1) run while they work on block n.
template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DA_THREADS, 1)
doc_attn_dq_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ CUtensorMap tmap_do, const __grid_constant__ CUtensorMap tmap_dq, const __grid_constant__ DocAttn p) {
    using S = DqSmem<D>;
    constexpr uint32_t TMEM_COLS = 512;     // S x2 [0,256)  dP [256,384)  dQ [384,384+D)
    constexpr uint32_t IDESC_S = make_idesc_f16_f32(128, 128, 0, 0);
    constexpr uint32_t IDESC_DQ = make_idesc_f16_f32(128, D, 0, 1);

    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = base;
    unsigned char* sDO = sQ + S::TILE;
    unsigned char* sK = sDO + S::TILE;
    unsigned char* sV = sK + S::STAGES * S::TILE;
    unsigned char* sOut = sV + S::STAGES * S::TILE;     // a patch for each owner warp
    float* again = reinterpret_cast<float*>(sOut + 16 * S::PATCH);     // [128]
    DaTable* table = reinterpret_cast<DaTable*>(again + 128);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + 1);
    uint64_t* q_full = bars;
    uint64_t* q_empty = bars + 1;
    uint64_t* k_full = bars + 2;       // STAGES
    uint64_t* k_empty = bars + 4;      // STAGES
    uint64_t* v_full = bars + 6;       // STAGES
    uint64_t* v_empty = bars + 8;      // STAGES
    uint64_t* s_full = bars + 10;      // 2
    uint64_t* ds_full = bars + 12;     // 2
    uint64_t* dp_full = bars + 14;
    uint64_t* dp_empty = bars + 15;
    uint64_t* acc_full = bars + 16;
    uint64_t* acc_empty = bars + 17;
    uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(bars + 18);

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int per_row = (p.tokens + 127) / 128, n_tiles = p.batch * per_row;
    const int group = p.heads / p.kv_heads;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&ds_full[i], 16);
        }
        mbar_init(dp_full, 1);
        mbar_init(dp_empty, 16);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_base_smem, TMEM_COLS);
        tmem_relinquish();
    }
    auto ranges = [&](int b, int t0, bool second) { return second ? Range{0, 0} : da_blocks<true>(p, b, t0, 128); };
    const int listed = da_plan_items(table, n_tiles, p.heads, per_row, 128, ranges);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = uniform(*tmem_base_smem);

    struct Item : DaItem {
        int n;
    };
    auto item_of = [&](int round, Item& m) {
        if (round < listed) static_cast<DaItem&>(m) = table->items[round];
        else if (listed < DA_LIST || !da_find_item(round, n_tiles, p.heads, per_row, 128, table, ranges, m)) return false;
        m.n = m.r0.end - m.r0.begin;
        return true;
    };

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            uint32_t it = 0, items = 0;
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                if (m.n == 0) continue;
                const int row = m.b * p.tokens, col = m.head * D, kcol = m.head / group * D;
                ok = mbar_wait(q_empty, (items++ & 1) ^ 1);
                if (!ok) break;
                mbar_arrive_expect_tx(q_full, 2 * S::TILE);
#pragma unroll
                for (int a = 0; a < D / 64; a++) {
                    tma_load_2d(sQ + a * 16384, &tmap_q, q_full, col + a * 64, row + m.t0);
                    tma_load_2d(sDO + a * 16384, &tmap_do, q_full, col + a * 64, row + m.t0);
                }
                for (int n = 0; n < m.n && ok; n++, it++) {
                    const int s = it % S::STAGES, y = row + (m.r0.begin + n) * 128;
                    const uint32_t par = ((it / S::STAGES) & 1) ^ 1;
                    ok = mbar_wait(&k_empty[s], par);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&k_full[s], S::TILE);
#pragma unroll
                    for (int a = 0; a < D / 64; a++) tma_load_2d(sK + s * S::TILE + a * 16384, &tmap_k, &k_full[s], kcol + a * 64, y);
                    ok = mbar_wait(&v_empty[s], par);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&v_full[s], S::TILE);
#pragma unroll
                    for (int a = 0; a < D / 64; a++) tma_load_2d(sV + s * S::TILE + a * 16384, &tmap_v, &v_full[s], kcol + a * 64, y);
                }
            }
            if (!ok) atomicExch(&g_doc_error, 21);
        }
    } else if (warp == 1) {
        {
            bool ok = true;
            const bool issuer = elect_one();
            const uint64_t q_desc = make_smem_desc_sw128(smem_u32(sQ), 16, 1024), do_desc = make_smem_desc_sw128(smem_u32(sDO), 16, 1024);
            const uint64_t k_desc = make_smem_desc_sw128(smem_u32(sK), 16, 1024), v_desc = make_smem_desc_sw128(smem_u32(sV), 16, 1024);
            const uint64_t k_col = make_smem_desc_sw128(smem_u32(sK), 16384, 1024);
            uint32_t it0 = 0, items = 0;
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                m.n = uniform(m.n);
                if (m.n == 0) continue;
                ok = mbar_wait(q_full, items & 1);
                for (int n = 0; n <= m.n && ok; n++) {
                    if (n < m.n) {
                        const uint32_t i = it0 + n;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&k_full[s], (i / S::STAGES) & 1);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint64_t kd = k_desc + (uint32_t)(s * (S::TILE >> 4)), vd = v_desc + (uint32_t)(s * (S::TILE >> 4));
                        if (issuer) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; kk++)      // S = Q K^T : [128 queries x 128 keys]
                                umma_f16_ss(tmem_base + sb * 128, q_desc + (kk >> 2) * 1024 + (kk & 3) * 2, kd + (kk >> 2) * 1024 + (kk & 3) * 2, IDESC_S,
                                            kk != 0 ? 1u : 0u);
                            umma_commit(&s_full[sb]);
                        }
                        ok = mbar_wait(&v_full[s], (i / S::STAGES) & 1) && mbar_wait(dp_empty, (i & 1) ^ 1);
                        if (!ok) break;
                        tcgen05_fence_after();
                        if (issuer) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; kk++)      // dP = dO V^T
                                umma_f16_ss(tmem_base + 256, do_desc + (kk >> 2) * 1024 + (kk & 3) * 2, vd + (kk >> 2) * 1024 + (kk & 3) * 2, IDESC_S,
                                            kk != 0 ? 1u : 0u);
                            umma_commit(dp_full);
                            umma_commit(&v_empty[s]);
                            if (n == m.n - 1) umma_commit(q_empty);
                        }
                    }
                    if (n >= 1) {
                        const uint32_t i = it0 + n - 1;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&ds_full[sb], (i >> 1) & 1);
                        if (ok && n == 1) ok = mbar_wait(acc_empty, (items & 1) ^ 1);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint64_t kd = k_col + (uint32_t)(s * (S::TILE >> 4));
                        if (issuer) {
#pragma unroll
                            for (int kk = 0; kk < 8; kk++)            // dQ += dS K : dS [128 q x 128 keys] in tensor memory, K [128 keys x d], d contiguous
                                umma_f16_ts(tmem_base + 384, tmem_base + sb * 128 + (kk >> 1) * 32 + (kk & 1) * 8, kd + kk * 128, IDESC_DQ,
                                            n != 1 || kk != 0 ? 1u : 0u);
                            umma_commit(&k_empty[s]);
                        }
                    }
                }
                if (ok && issuer) umma_commit(acc_full);
                it0 += m.n;
                items++;
            }
            if (!ok && issuer) atomicExch(&g_doc_error, 22);
        }
    } else {
        // ---------------- row owners: four threads per query, 32 of the 128 key columns each ----------------
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        const int r = quarter * 32 + lane, c0 = part * 32;
        const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16);
        unsigned char* const patch = sOut + (warp - 2) * S::PATCH;
        bool ok = true;
        uint32_t it0 = 0, items = 0;
        Item m = {}, following = {};
        int4 next_span = make_int4(0, 0, 0, 0);
        float next_lse = 0.0f, next_delta = 0.0f, next_slope = 0.0f;
        auto fetch = [&]() {
            const int qi = following.t0 + r;
            next_span = make_int4(0, 0x7fffffff, 0, 0);
            next_lse = next_delta = 0.0f;
            if (qi < p.tokens) {
                const int64_t at = ((int64_t)following.b * p.heads + following.head) * p.tokens + qi;
                next_span = p.spans[(int64_t)following.b * p.tokens + qi];
                next_lse = p.lse_in[at];
                next_delta = p.delta[at];
            }
            if (BIAS) next_slope = p.slopes[following.head];
        };
        bool have = item_of(0, following);
        if (have) fetch();
        for (int round = 1; have; round++) {
            m = following;
            const int qi = m.t0 + r;
            const bool live = qi < p.tokens;
            const int64_t row = (int64_t)m.b * p.tokens + qi;
            const int4 span = next_span;
            const float lse2 = next_lse * LOG2E, dlt = next_delta, slope2 = next_slope * LOG2E;
            have = item_of(round, following);           // the next item's row data travels while this one is worked on
            if (have) fetch();
            if (m.n == 0) {
                if (live) da_zero_row(p.dq + row * p.ld_dq + m.head * D + part * (D / 4), D / 4);
                continue;
            }
            const int lo = max(span.x, 0), hi = live ? min(span.y, p.tokens) : span.y;
            const bool ahead = BIAS && __any_sync(0xffffffffu, live && hi > qi + 1);
            for (int n = 0; n < m.n && ok; n++) {
                const uint32_t i = it0 + n;
                const int sb = i & 1, kbase = (m.r0.begin + n) * 128 + c0;
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[sb], (i >> 1) & 1) && mbar_wait(dp_full, i & 1));
                if (!ok) break;
                tcgen05_fence_after();
                const bool inner = lo <= kbase && hi >= kbase + 32 && (!BIAS || kbase + 31 <= qi || !ahead);
                const bool plain = __all_sync(0xffffffffu, inner);
                const float dist = (float)(kbase - qi);
                const float base = fmaf(slope2, dist, -lse2);
                const int from = lo - kbase, to = hi - kbase;
                const bool none_here = __all_sync(0xffffffffu, !(lo < kbase + 32 && hi > kbase));      // a corner that no row of the warp sees
                const uint32_t seen = span_bits(from, to);
                // 16 columns at a time: more do not fit the registers
#pragma unroll 1
                for (int c = 0; c < 2; c++) {
                    uint32_t w[8];
                    float2 x[8], g[8];
                    if (!none_here) {
                        tmem_ld_32x32b_x16(tm + sb * 128 + c0 + c * 16, reinterpret_cast<float*>(x));
                        tmem_ld_32x32b_x16(tm + 256 + c0 + c * 16, reinterpret_cast<float*>(g));
                        tmem_ld_wait();
                    }
                    if (c == 1) {
                        tcgen05_fence_before();
                        warp_arrive(dp_empty);
                    }
                    if (none_here) {
#pragma unroll
                        for (int e = 0; e < 8; e++) w[e] = 0;
                    } else {
                        bool near = true;
                        if (CAP) {
                            float wide = 0.0f;
#pragma unroll
                            for (int e = 0; e < 8; e++) wide = max3(wide, fabsf(x[e].x), fabsf(x[e].y));
                            near = __all_sync(0xffffffffu, wide * p.cap_in <= TANH_REACH);
                        }
                        auto step = [&](auto edge, auto reach) {
                            const float d0 = dist + (float)(c * 16);
                            Line bias(BIAS ? slope2 : 0.0f, BIAS ? fmaf(slope2, (float)(c * 16), base) : base);
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                float2 off = both(base), s, t;
                                if (BIAS) {
                                    if (edge)
                                        off = make_float2(fmaf(-slope2, fabsf(d0 + (float)(2 * e)), -lse2), fmaf(-slope2, fabsf(d0 + (float)(2 * e + 1)), -lse2));
                                    else
                                        off = bias.next(e);
                                }
                                if (CAP) {
                                    t = reach ? da_capped_near(x[e], p, both(0.0f)) : da_capped_far(x[e], p);
                                    s = __fadd2_rn(t, off);
                                } else {
                                    s = __ffma2_rn(x[e], both(p.scale_log2), off);
                                }
                                float2 de = __fmul2_rn(make_float2(fast_exp2(s.x), fast_exp2(s.y)), __fadd2_rn(g[e], both(-dlt)));
                                if (CAP) de = __fmul2_rn(de, __ffma2_rn(__fmul2_rn(t, both(p.cap_curve)), t, both(1.0f)));
                                if (edge) {
                                    const uint32_t bits = seen >> (c * 16 + 2 * e);
                                    if (!(bits & 1)) de.x = 0.0f;
                                    if (!(bits & 2)) de.y = 0.0f;
                                }
                                w[e] = da_half2(de.x, de.y);
                            }
                        };
                        if (near) {
                            if (plain) step(Flag<false>(), Flag<true>());
                            else step(Flag<true>(), Flag<true>());
                        } else {
                            step(Flag<true>(), Flag<false>());
                        }
                    }
                    tmem_st_32x32b_x8(tm + sb * 128 + c0 + c * 8, w);
                }
                tmem_st_wait();
                tcgen05_fence_before();
                warp_arrive(&ds_full[sb]);
            }
            it0 += m.n;
            if (ok) ok = mbar_wait(acc_full, items & 1);
            ok = __all_sync(0xffffffffu, ok);
            items++;
            const bool none = lo >= hi;
            float bad = 0.0f;
            if (ok) {
                tcgen05_fence_after();
#pragma unroll
                for (int c = 0; c < D / 4; c += 16) {
                    float2 a[8];
                    tmem_ld_32x32b_x16(tm + 384 + part * (D / 4) + c, reinterpret_cast<float*>(a));
                    tmem_ld_wait();
                    if (c + 16 == D / 4) {
                        tcgen05_fence_before();
                        warp_arrive(acc_empty);
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        bad = fmaf(a[i].x, 0.0f, fmaf(a[i].y, 0.0f, bad));
                        w[i] = none ? 0 : da_half2(a[i].x * p.scale, a[i].y * p.scale);
                    }
                    da_patch_free();
#pragma unroll
                    for (int i = 0; i < 2; i++) da_stage<16>(patch, lane, i, w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    da_patch_store(&tmap_dq, patch, m.head * D + part * (D / 4) + c, qi - lane, m.b, p.tokens);
                }
            }
            // evaluated again by the warps of the rows' first owners, after all owners' stores
            const bool redo_any = ok && live && !none && bad != 0.0f;
            if (barrier_any(1, 512, redo_any)) {
                if (part == 0) again[r] = 0.0f;
                asm volatile("bar.sync 1, 512;" ::: "memory");
                if (redo_any) again[r] = 1.0f;
                da_patch_written();
                asm volatile("bar.sync 1, 512;" ::: "memory");
                const bool redo = again[r] != 0.0f;
                if (part == 0 && __any_sync(0xffffffffu, redo)) da_mend_dq<D, CAP>(p, m.b, m.head, qi, lo, hi, redo);
                asm volatile("bar.sync 1, 512;" ::: "memory");
            }
        }
        da_patch_free();                                // the patch is read before the CTA's shared memory goes
        if (!ok && lane == 0) atomicExch(&g_doc_error, 23);
    }
    pdl_wait();                                          // what follows in the stream waits for this kernel and so for the dK / dV kernel too
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// ---- launches ------------------------------------------------------------------------------------------------------------

// The dynamic shared memory limit is an attribute of the kernel on a device: raised once for each.
template <typename K>
static int da_allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done, const char* where) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !(done.load() >> dev & 1))) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess && dev < 64) done.fetch_or((uint64_t)1 << dev);
    }
    if (e == cudaSuccess) return BRK_OK;
    set_cuda_error(e, where);
    return BRK_CUDA_ERROR;
}
// persistent: one CTA per SM walks the items
template <typename K, typename... Args>
static int da_launch(const char* name, K kernel, int64_t items, size_t smem, cudaStream_t st, const Args&... args) {
    const cudaError_t e = launch_pdl(kernel, (int)(items < sm_count() ? items : sm_count()), DA_THREADS, smem, st, args...);
    if (e != cudaSuccess) {
        set_cuda_error(e, name);
        return BRK_CUDA_ERROR;
    }
    return launch_status(name);
}

struct DocMaps {
    CUtensorMap q, k, v, d_out, q64, do64;      // operands
    CUtensorMap out, dq, dk, dv;                // results, [batch, tokens, columns]
};

template <int D, bool CAP, bool BIAS>
static int da_fwd(const DocMaps& t, const DocAttn& p, cudaStream_t st) {
    constexpr size_t smem = FwdSmem<D>::BYTES;
    static_assert(smem <= 232448, "the tile set must fit the 227 KB a CTA can have");
    static std::atomic<uint64_t> done{0};
    const int rc = da_allow_smem(doc_attn_fwd_kernel<D, CAP, BIAS>, smem, done, "doc_attn_fwd smem attribute");
    if (rc) return rc;
    return da_launch("doc_attn_fwd_kernel", doc_attn_fwd_kernel<D, CAP, BIAS>, (int64_t)p.batch * ((p.tokens + 255) / 256) * p.heads, smem, st, t.q, t.k, t.v, t.out, p);
}
template <int D, bool CAP, bool BIAS>
static int da_bwd(const DocMaps& t, const DocAttn& p, cudaStream_t st) {
    constexpr size_t smem_kv = DkvSmem<D>::BYTES, smem_q = DqSmem<D>::BYTES;
    static_assert(smem_kv <= 232448 && smem_q <= 232448, "the tile sets must fit the 227 KB a CTA can have");
    static std::atomic<uint64_t> done_kv{0}, done_q{0};
    int rc = da_allow_smem(doc_attn_dkv_kernel<D, CAP, BIAS>, smem_kv, done_kv, "doc_attn_dkv smem attribute");
    if (!rc) rc = da_allow_smem(doc_attn_dq_kernel<D, CAP, BIAS>, smem_q, done_q, "doc_attn_dq smem attribute");
    if (rc) return rc;
    const int64_t tiles = (int64_t)p.batch * ((p.tokens + 127) / 128);
    rc = da_launch("doc_attn_dkv_kernel", doc_attn_dkv_kernel<D, CAP, BIAS>, tiles * p.kv_heads, smem_kv, st, t.q64, t.k, t.v, t.do64, t.dk, t.dv, p);
    if (rc) return rc;
    return da_launch("doc_attn_dq_kernel", doc_attn_dq_kernel<D, CAP, BIAS>, tiles * p.heads, smem_q, st, t.q, t.k, t.v, t.d_out, t.dq, p);
}
template <int D, bool CAP>
static int da_run(bool forward, const DocMaps& t, const DocAttn& p, cudaStream_t st) {
    if (p.slopes) return forward ? da_fwd<D, CAP, true>(t, p, st) : da_bwd<D, CAP, true>(t, p, st);
    return forward ? da_fwd<D, CAP, false>(t, p, st) : da_bwd<D, CAP, false>(t, p, st);
}
static int da_dispatch(bool forward, int d, const DocMaps& t, const DocAttn& p, cudaStream_t st) {
    const bool cap = p.cap_log2 > 0.0f;
    if (d == 128) return cap ? da_run<128, true>(forward, t, p, st) : da_run<128, false>(forward, t, p, st);
    return cap ? da_run<64, true>(forward, t, p, st) : da_run<64, false>(forward, t, p, st);
}

// [batch, tokens, cols] fp16 with rows `ld` elements apart, boxes of 32 tokens x `box_cols` columns as da_stage lays them out
static bool da_result_map(CUtensorMap* out, void* base, int batch, int tokens, int64_t cols, int64_t ld, int box_cols) {
    const EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)tokens, (cuuint64_t)batch}, strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * (cuuint64_t)tokens};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, 32, 1}, one[3] = {1, 1, 1};
    return enc(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// sizes, strides and alignment that both directions share
static int da_check(const void* q, const void* k, const void* v, int64_t ld_q, int64_t ld_kv, const void* out, int64_t ld_out, const int32_t* spans, float cap,
                    int batch, int tokens, int heads, int kv_heads, int d) {
    if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || (d != 64 && d != 128)) return BRK_ATTR_ERROR;
    if (heads > 4096 || tokens > (1 << 22) || (int64_t)batch * tokens > (1 << 30)) return BRK_ATTR_ERROR;
    if ((int64_t)batch * ((tokens + 127) / 128) * heads > 0x7fffffff) return BRK_ATTR_ERROR;
    if (cap != 0.0f && !(cap >= 1e-6f && cap <= 1e4f)) return BRK_ATTR_ERROR;        // a NaN too; 1 / cap^2 stays finite
    if (ld_q % 8 != 0 || ld_kv % 8 != 0 || ld_out % 8 != 0 || ld_q < (int64_t)heads * d || ld_kv < (int64_t)kv_heads * d || ld_out < (int64_t)heads * d)
        return BRK_ATTR_ERROR;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(spans)) return BRK_ATTR_ERROR;
    return BRK_OK;
}
static DocAttn da_params(const void* q, const void* k, const void* v, int64_t ld_q, int64_t ld_kv, int64_t ld_out, const int32_t* spans, const float* slopes,
                         float cap, int batch, int tokens, int heads, int kv_heads, int d) {
    DocAttn p = {};
    p.q = (const __half*)q;
    p.k = (const __half*)k;
    p.v = (const __half*)v;
    p.ld_q = ld_q;
    p.ld_kv = ld_kv;
    p.ld_out = ld_out;
    p.spans = (const int4*)spans;
    p.slopes = slopes;
    p.batch = batch;
    p.tokens = tokens;
    p.heads = heads;
    p.kv_heads = kv_heads;
    const double scale = 1.0 / sqrt((double)d), log2e = 1.4426950408889634;
    p.scale = (float)scale;
    p.scale_log2 = (float)(scale * log2e);
    p.cap_log2 = (float)(cap * log2e);
    p.cap_in = cap > 0.0f ? (float)(scale / cap) : 0.0f;
    p.cap_curve = cap > 0.0f ? (float)(-1.0 / (cap * log2e * cap * log2e)) : 0.0f;
    const double tanh_poly[5] = {TANH_1, TANH_3, TANH_5, TANH_7, TANH_9};
    for (int i = 0; i < 5; i++) p.cap_poly[i] = (float)(tanh_poly[i] * cap * log2e);
    return p;
}

}  // namespace brk

using namespace brk;

extern "C" int brk_doc_attn_fwd(const void* q, const void* k, const void* v, int64_t ld_q, int64_t ld_kv, void* out, int64_t ld_out, float* lse,
                                const int32_t* spans, const float* slopes, float cap, int batch, int tokens, int heads, int kv_heads, int head_dim,
                                void* stream) {
    const int rc = da_check(q, k, v, ld_q, ld_kv, out, ld_out, spans, cap, batch, tokens, heads, kv_heads, head_dim);
    if (rc) return rc;
    if (batch == 0 || tokens == 0) return BRK_OK;
    if (!q || !k || !v || !spans) return BRK_INPUT_ERROR;
    if (!out) return BRK_OUTPUT_ERROR;
    DocAttn p = da_params(q, k, v, ld_q, ld_kv, ld_out, spans, slopes, cap, batch, tokens, heads, kv_heads, head_dim);
    p.out = (__half*)out;
    p.lse = lse;
    const uint64_t rows = (uint64_t)batch * tokens, qc = (uint64_t)heads * head_dim, kc = (uint64_t)kv_heads * head_dim;
    DocMaps t;
    if (!make_tmap_2d_f16(&t.q, q, rows, qc, (uint64_t)ld_q, 64, 128) || !make_tmap_2d_f16(&t.k, k, rows, kc, (uint64_t)ld_kv, 64, 128) ||
        !make_tmap_2d_f16(&t.v, v, rows, kc, (uint64_t)ld_kv, 64, 128) || !da_result_map(&t.out, out, batch, tokens, (int64_t)qc, ld_out, 32)) {
        set_error_message("brk_doc_attn_fwd: could not encode a tensor map");
        return BRK_CUDA_ERROR;
    }
    return da_dispatch(true, head_dim, t, p, (cudaStream_t)stream);
}

extern "C" size_t brk_doc_attn_bwd_workspace_bytes(int batch, int tokens, int heads) {
    if (batch <= 0 || tokens <= 0 || heads <= 0) return 0;
    return (size_t)batch * tokens * heads * sizeof(float);
}

extern "C" int brk_doc_attn_bwd(const void* q, const void* k, const void* v, int64_t ld_q, int64_t ld_kv, const void* out, const void* d_out, int64_t ld_out,
                                const float* lse, void* dq, int64_t ld_dq, void* dk, void* dv, int64_t ld_dkv, const int32_t* spans, const float* slopes,
                                float cap, int batch, int tokens, int heads, int kv_heads, int head_dim, void* workspace, size_t workspace_bytes,
                                void* stream) {
    int rc = da_check(q, k, v, ld_q, ld_kv, out, ld_out, spans, cap, batch, tokens, heads, kv_heads, head_dim);
    if (rc) return rc;
    if (ld_dq % 8 != 0 || ld_dkv % 8 != 0 || ld_dq < (int64_t)heads * head_dim || ld_dkv < (int64_t)kv_heads * head_dim) return BRK_ATTR_ERROR;
    if (!aligned16(d_out) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv)) return BRK_ATTR_ERROR;
    if (batch == 0 || tokens == 0) return BRK_OK;
    if (!q || !k || !v || !out || !d_out || !lse || !spans) return BRK_INPUT_ERROR;
    if (!dq || !dk || !dv) return BRK_OUTPUT_ERROR;
    if (!workspace || workspace_bytes < brk_doc_attn_bwd_workspace_bytes(batch, tokens, heads) || (reinterpret_cast<uintptr_t>(workspace) & 3)) return BRK_ATTR_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    DocAttn p = da_params(q, k, v, ld_q, ld_kv, ld_out, spans, slopes, cap, batch, tokens, heads, kv_heads, head_dim);
    p.d_out = (const __half*)d_out;
    p.lse_in = lse;
    p.delta = (const float*)workspace;
    p.dq = (__half*)dq;
    p.dk = (__half*)dk;
    p.dv = (__half*)dv;
    p.ld_dq = ld_dq;
    p.ld_dkv = ld_dkv;
    const uint64_t rows = (uint64_t)batch * tokens, qc = (uint64_t)heads * head_dim, kc = (uint64_t)kv_heads * head_dim;
    DocMaps t;
    if (!make_tmap_2d_f16(&t.q, q, rows, qc, (uint64_t)ld_q, 64, 128) || !make_tmap_2d_f16(&t.k, k, rows, kc, (uint64_t)ld_kv, 64, 128) ||
        !make_tmap_2d_f16(&t.v, v, rows, kc, (uint64_t)ld_kv, 64, 128) || !make_tmap_2d_f16(&t.d_out, d_out, rows, qc, (uint64_t)ld_out, 64, 128) ||
        !make_tmap_2d_f16(&t.q64, q, rows, qc, (uint64_t)ld_q, 64, DA_SUB) || !make_tmap_2d_f16(&t.do64, d_out, rows, qc, (uint64_t)ld_out, 64, DA_SUB) ||
        !da_result_map(&t.dq, dq, batch, tokens, (int64_t)qc, ld_dq, 16) || !da_result_map(&t.dk, dk, batch, tokens, (int64_t)kc, ld_dkv, head_dim / 4) ||
        !da_result_map(&t.dv, dv, batch, tokens, (int64_t)kc, ld_dkv, head_dim / 4)) {
        set_error_message("brk_doc_attn_bwd: could not encode a tensor map");
        return BRK_CUDA_ERROR;
    }
    const cudaError_t e = launch_pdl(doc_delta_kernel, batch * tokens, 256, 0, st, (const __half*)out, (const __half*)d_out, ld_out, (float*)workspace, tokens, heads, head_dim);
    if (e != cudaSuccess) {
        set_cuda_error(e, "doc_delta_kernel");
        return BRK_CUDA_ERROR;
    }
    rc = launch_status("doc_delta_kernel");
    if (rc) return rc;
    return da_dispatch(false, head_dim, t, p, st);
}

// Synchronous: non-zero if one of these kernels gave up on a bounded wait since the last query.
extern "C" int brk_doc_attn_status(void) {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, brk::g_doc_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(brk::g_doc_error, &zero, sizeof(int));
    return v;
}
