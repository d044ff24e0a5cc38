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
// finite and evaluate that row again in fp32 over its visible pairs alone, so a NaN or an infinity reaches exactly the
// rows that see it and costs nothing where there is none.
//
// Every mbarrier wait is bounded (see brk_ptx.cuh); a give-up raises g_doc_error.
#include <atomic>

#include "brk_attn.cuh"
#include "brk_common.cuh"
#include "brk_ptx.cuh"

namespace brk {

using namespace ptx;

__device__ int g_doc_error = 0;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int DA_THREADS = 64 + 256;        // producer warp, MMA warp, eight row-owner warps
constexpr int DA_SORT = 512;                // tiles whose order a CTA sorts; more are taken as they come

struct DocAttn {
    const __half *q, *k, *v;
    const int4* spans;                      // [batch, tokens]: lo, hi, qlo, qhi
    const float* slopes;                    // [heads] or null
    int64_t ld_q, ld_kv, ld_out;
    int batch, tokens, heads, kv_heads;
    float scale, scale_log2;                // 1/sqrt(d), times log2(e)
    float cap_log2, cap_in;                 // cap log2(e); 2 log2(e) / (sqrt(d) cap), so that exp2(cap_in q.k) = e^(2x/cap)
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

// Score of a raw product in log2 units without the bias, and with a cap the tanh's derivative.  tanh(u) = 1 - 2r with
// r = 1 / (1 + e^2u): absolute error about 1e-7 over the whole range, which at a cap of 50 is 1e-5 of the exponent (the
// hardware tanh's 2^-11 would be 0.02 of it).
template <bool CAP>
__device__ __forceinline__ float da_score(float raw, const DocAttn& p) {
    if (!CAP) return raw * p.scale_log2;
    const float r = __fdividef(1.0f, 1.0f + fast_exp2(raw * p.cap_in));
    return fmaf(-2.0f * p.cap_log2, r, p.cap_log2);
}
template <bool CAP>
__device__ __forceinline__ float da_score(float raw, const DocAttn& p, float& slope_of_tanh) {
    if (!CAP) {
        slope_of_tanh = 1.0f;
        return raw * p.scale_log2;
    }
    const float r = __fdividef(1.0f, 1.0f + fast_exp2(raw * p.cap_in));
    slope_of_tanh = 4.0f * r * (1.0f - r);
    return fmaf(-2.0f * p.cap_log2, r, p.cap_log2);
}

// ---- tiles ---------------------------------------------------------------------------------------------------------------

struct Range {
    int begin, end;
};
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
// direction, which evens out the totals without a counter in memory.  Every CTA sorts for itself (it needs two loads per
// tile); the table lives in shared memory.
struct DaTable {
    uint16_t order[DA_SORT];
    uint16_t weight[DA_SORT];
};
__device__ __forceinline__ bool da_item(int round, int n_tiles, int n_heads, const DaTable* table, bool sorted, int& tile, int& head) {
    const int64_t G = gridDim.x, c = blockIdx.x;
    const int64_t idx = round * G + ((round & 1) ? G - 1 - c : c);
    if (idx >= (int64_t)n_tiles * n_heads) return false;
    const int place = (int)(idx / n_heads);
    tile = sorted ? table->order[place] : n_tiles - 1 - place;
    head = (int)(idx % n_heads);
    return true;
}
// weight(tile) for all tiles, then the rank of each: heavier first, ties by number.  All threads of the CTA.
template <typename W>
__device__ __forceinline__ void da_sort(DaTable* table, int n_tiles, W weight) {
    for (int i = threadIdx.x; i < n_tiles; i += DA_THREADS) table->weight[i] = (uint16_t)min(weight(i), 65535);
    __syncthreads();
    for (int i = threadIdx.x; i < n_tiles; i += DA_THREADS) {
        const int w = table->weight[i];
        int rank = 0;
        for (int j = 0; j < n_tiles; j++) rank += table->weight[j] > w || (table->weight[j] == w && j < i);
        table->order[rank] = (uint16_t)i;
    }
}

// ---- rows evaluated again without the tensor core (see the top) ------------------------------------------------------------

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
template <int D, bool CAP>
__device__ float da_log2_score(const DocAttn& p, int b, int h, int i, int j, float& dt) {
    const int kh = h / (p.heads / p.kv_heads);
    const __half* q = p.q + ((int64_t)b * p.tokens + i) * p.ld_q + h * D;
    const __half* k = p.k + ((int64_t)b * p.tokens + j) * p.ld_kv + kh * D;
    float s = da_score<CAP>(da_dot<D>(q, k), p, dt);
    if (p.slopes) s -= p.slopes[h] * LOG2E * fabsf((float)(i - j));
    return s;
}
template <int D, bool CAP>
__device__ __noinline__ void da_out_row(const DocAttn& p, int b, int h, int i, int lo, int hi, float lse2) {
    const int kh = h / (p.heads / p.kv_heads);
    __half* o = p.out + ((int64_t)b * p.tokens + i) * p.ld_out + h * D;
    for (int c = 0; c < D; c += 32) {
        float acc[32] = {};
        for (int j = lo; j < hi; j++) {
            float dt;
            const float w = fast_exp2(da_log2_score<D, CAP>(p, b, h, i, j, dt) - lse2);
            const __half* v = p.v + ((int64_t)b * p.tokens + j) * p.ld_kv + kh * D + c;
#pragma unroll
            for (int e = 0; e < 32; e++) acc[e] = fmaf(w, __half2float(v[e]), acc[e]);
        }
        for (int e = 0; e < 32; e++) o[c + e] = __float2half_rn(acc[e]);
    }
}
// P and dS of one visible pair
template <int D, bool CAP>
__device__ float da_pair(const DocAttn& p, int b, int h, int i, int j, float& ds) {
    const int kh = h / (p.heads / p.kv_heads);
    const int64_t at = ((int64_t)b * p.heads + h) * p.tokens + i;
    float dt;
    const float w = fast_exp2(da_log2_score<D, CAP>(p, b, h, i, j, dt) - p.lse_in[at] * LOG2E);
    const float dp = da_dot<D>(p.d_out + ((int64_t)b * p.tokens + i) * p.ld_out + h * D, p.v + ((int64_t)b * p.tokens + j) * p.ld_kv + kh * D);
    ds = w * (dp - p.delta[at]) * dt;
    return w;
}
template <int D, bool CAP>
__device__ __noinline__ void da_dq_row(const DocAttn& p, int b, int h, int i, int lo, int hi) {
    const int kh = h / (p.heads / p.kv_heads);
    __half* o = p.dq + ((int64_t)b * p.tokens + i) * p.ld_dq + h * D;
    for (int c = 0; c < D; c += 32) {
        float acc[32] = {};
        for (int j = lo; j < hi; j++) {
            float ds;
            da_pair<D, CAP>(p, b, h, i, j, ds);
            const __half* k = p.k + ((int64_t)b * p.tokens + j) * p.ld_kv + kh * D + c;
#pragma unroll
            for (int e = 0; e < 32; e++) acc[e] = fmaf(ds, __half2float(k[e]), acc[e]);
        }
        for (int e = 0; e < 32; e++) o[c + e] = __float2half_rn(acc[e] * p.scale);
    }
}
template <int D, bool CAP>
__device__ __noinline__ void da_dkv_row(const DocAttn& p, int b, int kh, int j, int qlo, int qhi) {
    const int group = p.heads / p.kv_heads;
    const int64_t at = ((int64_t)b * p.tokens + j) * p.ld_dkv + kh * D;
    for (int c = 0; c < D; c += 32) {
        float ak[32] = {}, av[32] = {};
        for (int h = kh * group; h < (kh + 1) * group; h++)
            for (int i = qlo; i < qhi; i++) {
                float ds;
                const float w = da_pair<D, CAP>(p, b, h, i, j, ds);
                const __half* q = p.q + ((int64_t)b * p.tokens + i) * p.ld_q + h * D + c;
                const __half* g = p.d_out + ((int64_t)b * p.tokens + i) * p.ld_out + h * D + c;
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    ak[e] = fmaf(ds, __half2float(q[e]), ak[e]);
                    av[e] = fmaf(w, __half2float(g[e]), av[e]);
                }
            }
        for (int e = 0; e < 32; e++) {
            p.dk[at + c + e] = __float2half_rn(ak[e] * p.scale);
            p.dv[at + c + e] = __float2half_rn(av[e]);
        }
    }
}

__device__ __forceinline__ void da_zero_row(__half* row, int d) {
    for (int e = 0; e < d; e += 8) *reinterpret_cast<uint4*>(row + e) = make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint32_t da_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ==========================================================================================================================
// forward
//
// An item is 256 queries of one head: two tiles of 128 that share the K and V tiles.  Each tile has its own score columns
// in tensor memory, its own output accumulator and its own four softmax warps, one thread per query.  While one tile's
// warps exponentiate, the tensor core works for the other: S0 S1 | PV0 S0' | PV1 S1' | ...  Probabilities go back to
// tensor memory, over the scores they came from, as the A operand of P V: they never pass through shared memory, whose
// bandwidth the two operands of Q K^T already need.  A tile's next scores may be issued right behind its P V without a
// wait, since the tensor core works off its instructions in order.
// The running maximum is lazy: probabilities are taken relative to a reference that moves (and the accumulator is
// rescaled) only when the true maximum has run ahead of it by 2^8, so that P stays far inside fp16; fp16 and not fp32
// because it is the tensor core's operand type: 2^-11 of each probability, the same as V's own rounding.
// ==========================================================================================================================
template <int D>
struct FwdSmem {
    static constexpr uint32_t TILE = 128 * D * 2;
    static constexpr int STAGES = 2;                    // of K and of V each
    static constexpr size_t BYTES = 1024 + TILE * (2 + 2 * STAGES) + sizeof(DaTable) + 256;
};

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DA_THREADS, 1)
doc_attn_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                    const __grid_constant__ DocAttn p) {
    using S = FwdSmem<D>;
    constexpr uint32_t TMEM_COLS = 512;                 // S0 [0,128)  S1 [128,256)  O0 [256,256+D)  O1 [256+D,256+2D)
    constexpr uint32_t IDESC_S = make_idesc_f16_f32(128, 128, 0, 0);
    constexpr uint32_t IDESC_PV = make_idesc_f16_f32(128, D, 0, 1);
    constexpr float RESCALE_STEP = 8.0f;                // log2 units the row maximum may run ahead of the reference

    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = base;                           // two tiles
    unsigned char* sK = sQ + 2 * S::TILE;
    unsigned char* sV = sK + S::STAGES * S::TILE;
    DaTable* table = reinterpret_cast<DaTable*>(sV + S::STAGES * S::TILE);
    uint64_t* bars = reinterpret_cast<uint64_t*>(table + 1);
    uint64_t* q_full = bars;                 // 2 (per tile)
    uint64_t* q_empty = bars + 2;            // 2
    uint64_t* k_full = bars + 4;             // STAGES
    uint64_t* k_empty = bars + 6;
    uint64_t* v_full = bars + 8;
    uint64_t* v_empty = bars + 10;
    uint64_t* s_full = bars + 12;            // 2 (per tile)
    uint64_t* p_full = bars + 14;            // 2
    uint64_t* o_done = bars + 16;            // 2: a P V product of the tile is complete
    uint64_t* o_empty = bars + 18;           // 2: the tile's output has been read
    uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(bars + 20);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = (p.tokens + 255) / 256, n_pairs = p.batch * per_row;
    const bool sorted = n_pairs <= DA_SORT;

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; t++) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&k_full[t], 1);
            mbar_init(&k_empty[t], 1);
            mbar_init(&v_full[t], 1);
            mbar_init(&v_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 128);
            mbar_init(&o_done[t], 1);
            mbar_init(&o_empty[t], 128);
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
    if (sorted)
        da_sort(table, n_pairs, [&](int i) {
            const int b = i / per_row, t0 = (i % per_row) * 256;
            const Range r0 = da_blocks<true>(p, b, t0, 128), r1 = da_blocks<true>(p, b, t0 + 128, 128);
            return r0.end - r0.begin + r1.end - r1.begin;
        });
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_base_smem;
    const int group = p.heads / p.kv_heads;

    struct Item {
        int b, t0, head;
        Range r[2];          // key blocks of the two tiles
        int first, n;        // the blocks that either needs
    };
    auto item_of = [&](int round, Item& m) {
        int pair;
        if (!da_item(round, n_pairs, p.heads, table, sorted, pair, m.head)) return false;
        m.b = pair / per_row;
        m.t0 = (pair % per_row) * 256;
        m.r[0] = da_blocks<true>(p, m.b, m.t0, 128);
        m.r[1] = da_blocks<true>(p, m.b, m.t0 + 128, 128);
        const bool has0 = m.r[0].end > m.r[0].begin, has1 = m.r[1].end > m.r[1].begin;
        m.first = has0 ? (has1 ? min(m.r[0].begin, m.r[1].begin) : m.r[0].begin) : m.r[1].begin;
        m.n = max(m.r[0].end, m.r[1].end) - m.first;
        return true;
    };

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            bool ok = true;
            uint32_t it = 0, q_count[2] = {0, 0};
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                const int row = m.b * p.tokens, col = m.head * D, kcol = m.head / group * D;
                for (int t = 0; t < 2 && ok; t++) {
                    if (m.r[t].end == m.r[t].begin) continue;
                    ok = mbar_wait(&q_empty[t], (q_count[t]++ & 1) ^ 1);        // the previous item's scores no longer read Q
                    if (!ok) break;
                    mbar_arrive_expect_tx(&q_full[t], S::TILE);
#pragma unroll
                    for (int a = 0; a < D / 64; a++) tma_load_2d(sQ + t * S::TILE + a * 16384, &tmap_q, &q_full[t], col + a * 64, row + m.t0 + t * 128);
                }
                for (int n = 0; n < m.n && ok; n++, it++) {
                    const int s = it % S::STAGES, y = row + (m.first + n) * 128;
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
            if (!ok) atomicExch(&g_doc_error, 1);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            bool ok = true;
            uint32_t it = 0, q_count[2] = {0, 0}, p_count[2] = {0, 0};        // blocks, and per tile: items, blocks
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                for (int n = -1; n < m.n && ok; n++) {
                    const int vs = (it + n) % S::STAGES, ks = (it + n + 1) % S::STAGES;        // n == -1 uses no V
                    const bool more = n + 1 < m.n;
                    if (n >= 0) ok = mbar_wait(&v_full[vs], ((it + n) / S::STAGES) & 1);
                    if (ok && more) ok = mbar_wait(&k_full[ks], ((it + n + 1) / S::STAGES) & 1);
                    for (int t = 0; t < 2 && ok; t++) {
                        const int blk = m.first + n;
                        if (n >= 0 && blk >= m.r[t].begin && blk < m.r[t].end) {
                            ok = mbar_wait(&p_full[t], p_count[t] & 1);
                            if (ok && blk == m.r[t].begin) ok = mbar_wait(&o_empty[t], (q_count[t] & 1));      // count is one ahead: this item's scores are out
                            if (!ok) break;
                            tcgen05_fence_after();
                            const uint32_t v_addr = smem_u32(sV + vs * S::TILE);
#pragma unroll
                            for (int kk = 0; kk < 8; kk++)        // A = P [128 q x 128 keys] in tensor memory, B = V [128 keys x D], d contiguous
                                umma_f16_ts(tmem_base + 256 + t * D, tmem_base + t * 128 + kk * 8, make_smem_desc_sw128(v_addr + kk * 2048, 16384, 1024), IDESC_PV,
                                            (blk != m.r[t].begin || kk != 0) ? 1u : 0u);
                            umma_commit(&o_done[t]);
                            p_count[t]++;
                        }
                        if (more && blk + 1 >= m.r[t].begin && blk + 1 < m.r[t].end) {
                            if (blk + 1 == m.r[t].begin) {
                                ok = mbar_wait(&q_full[t], q_count[t]++ & 1);
                                if (!ok) break;
                            }
                            tcgen05_fence_after();
                            const uint32_t q_addr = smem_u32(sQ + t * S::TILE), k_addr = smem_u32(sK + ks * S::TILE);
#pragma unroll
                            for (int kk = 0; kk < D / 16; kk++) {
                                const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                                umma_f16_ss(tmem_base + t * 128, make_smem_desc_sw128(q_addr + off, 16, 1024), make_smem_desc_sw128(k_addr + off, 16, 1024), IDESC_S,
                                            kk != 0 ? 1u : 0u);
                            }
                            umma_commit(&s_full[t]);
                            if (blk + 2 == m.r[t].end) umma_commit(&q_empty[t]);
                        }
                    }
                    if (!ok) break;
                    if (n >= 0) umma_commit(&v_empty[vs]);
                    if (more) umma_commit(&k_empty[ks]);
                }
                it += m.n;
            }
            if (!ok) atomicExch(&g_doc_error, 2);
        }
    } else {
        // ---------------- softmax / epilogue: one thread per query of the tile ----------------
        const int t = (warp - 2) >> 2;                  // tile: warps 2-5 and 6-9
        const int quarter = warp & 3;                   // a warp reaches tensor-memory lanes 32 * (warp % 4) ..
        const int r = quarter * 32 + lane;
        const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tm_s = tm + t * 128, tm_o = tm + 256 + t * D;
        bool ok = true;
        uint32_t it = 0;
        Item m;
        for (int round = 0; item_of(round, m); round++) {
            const int qi = m.t0 + t * 128 + r;
            const bool live = qi < p.tokens;
            const int64_t row = (int64_t)m.b * p.tokens + qi;
            int4 span = make_int4(0, 0x7fffffff, 0, 0);             // rows behind the sequence never force the masked path
            if (live) span = p.spans[row];
            const int lo = max(span.x, 0), hi = live ? min(span.y, p.tokens) : span.y;
            if (m.r[t].end == m.r[t].begin) {
                if (live) {
                    da_zero_row(p.out + row * p.ld_out + m.head * D, D);
                    if (p.lse) p.lse[((int64_t)m.b * p.heads + m.head) * p.tokens + qi] = 0.0f;
                }
                continue;
            }
            const float slope2 = BIAS ? p.slopes[m.head] * LOG2E : 0.0f;
            const bool ahead = BIAS && __any_sync(0xffffffffu, live && hi > qi + 1);      // some row sees keys behind itself: the prompt's
            float m_ref = -INFINITY, l = 0.0f;
            for (int blk = m.r[t].begin; blk < m.r[t].end; blk++, it++) {
                if (ok) ok = mbar_wait(&s_full[t], it & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) continue;
                tcgen05_fence_after();
                const int kbase = blk * 128;
                const bool full = __all_sync(0xffffffffu, lo <= kbase && hi >= kbase + 128);
                const bool past = !ahead || __all_sync(0xffffffffu, kbase + 127 <= qi);
                const float base = slope2 * (float)(kbase - qi), dist = (float)(kbase - qi);
                float x[128];
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t v[32];
                    tmem_ld_32x32b_x32(tm_s + c * 32, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const int k = c * 32 + e;
                        float s = da_score<CAP>(__uint_as_float(v[e]), p);
                        if (BIAS) {
                            if (past)
                                s += fmaf(slope2, (float)k, base);
                            else
                                s = fmaf(-slope2, fabsf(dist + (float)k), s);
                        }
                        if (!full) s = (kbase + k >= lo && kbase + k < hi) ? s : -INFINITY;
                        x[k] = s;
                        top = fmaxf(top, s);
                    }
                }
                const bool move = top > m_ref + RESCALE_STEP;        // also the row's first visible key (m_ref = -inf)
                float factor = 1.0f;
                if (move) {
                    factor = m_ref == -INFINITY ? 0.0f : fast_exp2(m_ref - top);
                    m_ref = top;
                    l *= factor;
                }
                if (blk > m.r[t].begin && __any_sync(0xffffffffu, move)) {
                    // the accumulator may only be touched between two P V products: wait for the previous one
                    ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (it - 1) & 1));
                    if (!ok) continue;
                    tcgen05_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t v[32];
                        tmem_ld_32x32b_x32(tm_o + c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * factor);
                        tmem_st_32x32b_x32(tm_o + c, v);
                    }
                }
                const float ref = m_ref == -INFINITY ? 0.0f : m_ref;        // nothing visible yet: every exponential is 0
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t w[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const float p0 = fast_exp2(x[c * 64 + 2 * e] - ref), p1 = fast_exp2(x[c * 64 + 2 * e + 1] - ref);
                        l += p0 + p1;
                        w[e] = da_half2(p0, p1);
                    }
                    tmem_st_32x32b_x32(tm_s + c * 32, w);
                }
                tmem_st_wait();
                tcgen05_fence_before();
                mbar_arrive(&p_full[t]);
            }
            // epilogue: O / l -> fp16, token-major; log-sum-exp for the backward
            if (ok) ok = mbar_wait(&o_done[t], (it - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            tcgen05_fence_after();
            const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);        // a NaN stays one
            const float lse2 = m_ref + __log2f(l);
            __half* o = p.out + row * p.ld_out + m.head * D;
            const bool none = lo >= hi;
            float bad = 0.0f;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(tm_o + c, v);
                tmem_ld_wait();
                if (live) {
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        Vec<__half> w;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float a = __uint_as_float(v[g * 8 + e]);
                            bad = fmaf(a, 0.0f, bad);
                            w.v[e] = none ? 0.0f : a * inv;
                        }
                        w.store(o + c + g * 8);
                    }
                }
            }
            tcgen05_fence_before();
            mbar_arrive(&o_empty[t]);
            if (live) {
                if (p.lse) p.lse[((int64_t)m.b * p.heads + m.head) * p.tokens + qi] = none ? 0.0f : lse2 * LN2;
                if (bad != 0.0f && !none && fabsf(lse2) < INFINITY) da_out_row<D, CAP>(p, m.b, m.head, qi, lo, hi, lse2);
            }
        }
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
// Two threads share a row (warps w and w + 4 own the same 32 tensor-memory lanes and split the columns): one warp per
// scheduler could not hide the latency of its own loads and exponentials.  P and dS return to tensor memory over the
// scores they came from, as A operands; each half of the columns stays inside its own half of the region, so neither
// owner overwrites what the other has yet to read.  They are rounded to fp16 there, as operands have to be.
// ==========================================================================================================================

// delta_i = sum_d dO_id O_id per query and head: d / 8 neighbouring lanes own one head of one row
__global__ void __launch_bounds__(256)
doc_delta_kernel(const __half* out, const __half* dout, int64_t ld, float* delta, int batch, int tokens, int heads, int d) {
    const int lanes = d >> 3;
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t grp = t / lanes;
    const int part = (int)(t % lanes);
    const bool live = grp < (int64_t)batch * tokens * heads;
    const int h = (int)(grp % heads);
    const int64_t row = grp / heads;
    float s = 0.0f;
    if (live) {
        Vec<__half> a, c;
        a.load(out + row * ld + (int64_t)h * d + part * 8);
        c.load(dout + row * ld + (int64_t)h * d + part * 8);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf(a.v[e], c.v[e], s);
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (live && part == 0) delta[((row / tokens) * heads + h) * tokens + row % tokens] = s;
}

constexpr int DA_SUB = 64;                  // queries per step of the dK / dV kernel
constexpr uint32_t DA_SUB_ATOM = DA_SUB * 128;

template <int D>
struct DkvSmem {
    static constexpr uint32_t KV = 128 * D * 2, SUB = DA_SUB * D * 2;
    static constexpr int STAGES = 4;
    static constexpr size_t BYTES = 1024 + 2 * KV + 2 * STAGES * SUB + 2 * 2 * DA_SUB * sizeof(float) + sizeof(DaTable) + 256;
};

// Transposed scores S^T = K Q^T and dP^T = V dO^T (a row owner is a key), so that P^T and dS^T are the A operands of
// dV += P^T dO and dK += dS^T Q as they stand; the 64 queries' lse and delta of a step come from shared memory.  With
// shared key heads the walk goes over all query heads of the group, and the sum over them stays in the accumulators.
template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DA_THREADS, 1)
doc_attn_dkv_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                    const __grid_constant__ CUtensorMap tmap_do, const __grid_constant__ DocAttn p) {
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
    float* stat = reinterpret_cast<float*>(sDO + S::STAGES * S::SUB);       // [2][lse2 x 64 | delta x 64]
    DaTable* table = reinterpret_cast<DaTable*>(stat + 2 * 2 * DA_SUB);
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

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = (p.tokens + 127) / 128, n_tiles = p.batch * per_row;
    const int group = p.heads / p.kv_heads;
    const bool sorted = n_tiles <= DA_SORT;

    if (threadIdx.x == 0) {
        mbar_init(kv_full, 1);
        mbar_init(kv_empty, 1);
        for (int i = 0; i < S::STAGES; i++) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 256);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 256);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_base_smem, TMEM_COLS);
        tmem_relinquish();
    }
    if (sorted)
        da_sort(table, n_tiles, [&](int i) {
            const Range r = da_blocks<false>(p, i / per_row, (i % per_row) * 128, DA_SUB);
            return r.end - r.begin;
        });
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_base_smem;

    struct Item {
        int b, t0, head;       // head: of the keys
        Range r;               // 64-query blocks
        int n;                 // steps: blocks times query heads of the group
    };
    auto item_of = [&](int round, Item& m) {
        int tile;
        if (!da_item(round, n_tiles, p.kv_heads, table, sorted, tile, m.head)) return false;
        m.b = tile / per_row;
        m.t0 = (tile % per_row) * 128;
        m.r = da_blocks<false>(p, m.b, m.t0, DA_SUB);
        m.n = (m.r.end - m.r.begin) * group;
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
                int blk = m.r.begin, col = m.head * group * D;
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
                    if (++blk == m.r.end) {
                        blk = m.r.begin;
                        col += D;
                    }
                }
            }
            if (!ok) atomicExch(&g_doc_error, 11);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
            uint32_t it0 = 0, items = 0;
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
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
                        const uint32_t q_addr = smem_u32(sQ + s * S::SUB), do_addr = smem_u32(sDO + s * S::SUB);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++)      // S^T = K Q^T : [128 keys x 64 queries]
                            umma_f16_ss(tmem_base + sb * DA_SUB, make_smem_desc_sw128(k_addr + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                                        make_smem_desc_sw128(q_addr + (kk >> 2) * DA_SUB_ATOM + (kk & 3) * 32, 16, 1024), IDESC_ST, kk != 0 ? 1u : 0u);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++)      // dP^T = V dO^T
                            umma_f16_ss(tmem_base + 128 + sb * DA_SUB, make_smem_desc_sw128(v_addr + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                                        make_smem_desc_sw128(do_addr + (kk >> 2) * DA_SUB_ATOM + (kk & 3) * 32, 16, 1024), IDESC_ST, kk != 0 ? 1u : 0u);
                        umma_commit(&s_full[sb]);
                        if (n == m.n - 1) umma_commit(kv_empty);       // last products of the item that read K / V
                    }
                    if (n >= 1) {
                        const uint32_t i = it0 + n - 1;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&p_full[sb], (i >> 1) & 1);
                        if (ok && n == 1) ok = mbar_wait(acc_empty, (items & 1) ^ 1);      // the previous item's dV / dK have been read
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint32_t q_addr = smem_u32(sQ + s * S::SUB), do_addr = smem_u32(sDO + s * S::SUB);
#pragma unroll
                        for (int kk = 0; kk < DA_SUB / 16; kk++)      // dV += P^T dO (contraction over the 64 queries)
                            umma_f16_ts(tmem_base + 256, tmem_base + sb * DA_SUB + (kk >> 1) * 32 + (kk & 1) * 8,
                                        make_smem_desc_sw128(do_addr + kk * 2048, DA_SUB_ATOM, 1024), IDESC_ACC, (n != 1 || kk != 0) ? 1u : 0u);
#pragma unroll
                        for (int kk = 0; kk < DA_SUB / 16; kk++)      // dK += dS^T Q
                            umma_f16_ts(tmem_base + 256 + D, tmem_base + 128 + sb * DA_SUB + (kk >> 1) * 32 + (kk & 1) * 8,
                                        make_smem_desc_sw128(q_addr + kk * 2048, DA_SUB_ATOM, 1024), IDESC_ACC, (n != 1 || kk != 0) ? 1u : 0u);
                        umma_commit(&q_empty[s]);
                    }
                }
                if (ok) umma_commit(acc_full);
                it0 += m.n;
                items++;
            }
            if (!ok) atomicExch(&g_doc_error, 12);
        }
    } else {
        // ---------------- row owners: two threads per key, 32 of the 64 query columns each ----------------
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int r = quarter * 32 + lane, c0 = half * 32;
        const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16);
        bool ok = true;
        uint32_t it0 = 0, items = 0;
        Item m;
        for (int round = 0; item_of(round, m); round++) {
            const int kj = m.t0 + r;
            const bool live = kj < p.tokens;
            const int64_t row = (int64_t)m.b * p.tokens + kj;
            __half* dkrow = p.dk + row * p.ld_dkv + m.head * D;
            __half* dvrow = p.dv + row * p.ld_dkv + m.head * D;
            if (m.n == 0) {
                if (half == 0 && live) {
                    da_zero_row(dkrow, D);
                    da_zero_row(dvrow, D);
                }
                continue;
            }
            int4 span = make_int4(0, 0, 0, 0x7fffffff);              // rows behind the sequence never force the masked path
            if (live) span = p.spans[row];
            const int qlo = max(span.z, 0), qhi = live ? min(span.w, p.tokens) : span.w;
            int blk = m.r.begin, h = m.head * group;
            for (int n = 0; n < m.n; n++) {
                const uint32_t i = it0 + n;
                const int sb = i & 1, q0 = blk * DA_SUB;
                const float slope2 = BIAS ? p.slopes[h] * LOG2E : 0.0f;
                if (half == 0) {
                    // the step's 64 log-sum-exps (log2 units, with the query's share of the bias) and 64 deltas
                    const int c = r & 63, qi = q0 + c;
                    const int64_t at = ((int64_t)m.b * p.heads + h) * p.tokens + qi;
                    float v = 0.0f;
                    if (qi < p.tokens) v = r < 64 ? fmaf(p.lse_in[at], LOG2E, slope2 * (float)c) : p.delta[at];
                    stat[sb * 128 + r] = v;
                }
                // orders this step's writes after every thread's reads two steps ago; every owner reaches it in every step,
                // also one whose bounded wait gave up (it only skips the work)
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (ok) ok = mbar_wait(&s_full[sb], (i >> 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (ok) {
                    tcgen05_fence_after();
                    const float* lse2 = stat + sb * 128 + c0;
                    const float* dlt = lse2 + 64;
                    const bool full = __all_sync(0xffffffffu, qlo <= q0 + c0 && qhi >= q0 + c0 + 32);
                    const bool past = !BIAS || __all_sync(0xffffffffu, kj <= q0 + c0);
                    const float bias = slope2 * (float)(kj - q0);          // minus slope * (i - q0), which lse2 holds
                    uint32_t sv[32], dv[32], wp[16], wd[16];
                    tmem_ld_32x32b_x32(tm + sb * DA_SUB + c0, sv);
                    tmem_ld_32x32b_x32(tm + 128 + sb * DA_SUB + c0, dv);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float pe[2], de[2];
#pragma unroll
                        for (int f = 0; f < 2; f++) {
                            const int qi = q0 + c0 + e + f;
                            float dt;
                            float s = da_score<CAP>(__uint_as_float(sv[e + f]), p, dt);
                            s += bias - lse2[e + f];
                            if (BIAS && !past) s += fminf(0.0f, 2.0f * slope2 * (float)(qi - kj));        // a key ahead of the query: -slope (j - i)
                            pe[f] = fast_exp2(s);
                            de[f] = pe[f] * (__uint_as_float(dv[e + f]) - dlt[e + f]);
                            if (CAP) de[f] *= dt;
                            if (!full && !(qlo <= qi && qi < qhi)) pe[f] = de[f] = 0.0f;
                        }
                        wp[e >> 1] = da_half2(pe[0], pe[1]);
                        wd[e >> 1] = da_half2(de[0], de[1]);
                    }
                    tmem_st_32x32b_x16(tm + sb * DA_SUB + c0, wp);
                    tmem_st_32x32b_x16(tm + 128 + sb * DA_SUB + c0, wd);
                    tmem_st_wait();
                    tcgen05_fence_before();
                    mbar_arrive(&p_full[sb]);
                }
                if (++blk == m.r.end) {
                    blk = m.r.begin;
                    h++;
                }
            }
            it0 += m.n;
            if (ok) ok = mbar_wait(acc_full, items & 1);
            ok = __all_sync(0xffffffffu, ok);
            items++;
            float bad = 0.0f;
            const bool none = qlo >= qhi;
            if (ok) {
                tcgen05_fence_after();
#pragma unroll 1
                for (int d0 = half * (D / 2); d0 < (half + 1) * (D / 2); d0 += 32) {
                    uint32_t a[32], c[32];
                    tmem_ld_32x32b_x32(tm + 256 + d0, a);
                    tmem_ld_32x32b_x32(tm + 256 + D + d0, c);
                    tmem_ld_wait();
                    if (live) {
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            Vec<__half> o1, o2;
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const float x = __uint_as_float(a[g * 8 + e]), y = __uint_as_float(c[g * 8 + e]);
                                bad = fmaf(x, 0.0f, fmaf(y, 0.0f, bad));
                                o1.v[e] = none ? 0.0f : x;
                                o2.v[e] = none ? 0.0f : y * p.scale;
                            }
                            o1.store(dvrow + d0 + g * 8);
                            o2.store(dkrow + d0 + g * 8);
                        }
                    }
                }
                tcgen05_fence_before();
                mbar_arrive(acc_empty);            // the accumulators may take the next item's first products
            }
            // Evaluated again by the row's first owner, after both owners' stores (the barrier orders them).
            stat[half * 128 + r] = bad;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (half == 0 && live && !none && (stat[r] != 0.0f || stat[128 + r] != 0.0f)) da_dkv_row<D, CAP>(p, m.b, m.head, kj, qlo, qhi);
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
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
    static constexpr size_t BYTES = 1024 + 2 * TILE + 2 * STAGES * TILE + 2 * 128 * sizeof(float) + sizeof(DaTable) + 256;
};

// S = Q K^T (two buffers), dP = dO V^T (one), dQ += dS K over blocks of 128 keys.  dS goes over the scores it came from,
// so dP's buffer is free as soon as the owners have read it: S(n+1) and dP(n+1) run while they work on block n.
template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(DA_THREADS, 1)
doc_attn_dq_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ CUtensorMap tmap_do, const __grid_constant__ DocAttn p) {
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
    float* again = reinterpret_cast<float*>(sV + S::STAGES * S::TILE);     // [2 owners][128]
    DaTable* table = reinterpret_cast<DaTable*>(again + 2 * 128);
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

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = (p.tokens + 127) / 128, n_tiles = p.batch * per_row;
    const int group = p.heads / p.kv_heads;
    const bool sorted = n_tiles <= DA_SORT;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&ds_full[i], 256);
        }
        mbar_init(dp_full, 1);
        mbar_init(dp_empty, 256);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 256);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_base_smem, TMEM_COLS);
        tmem_relinquish();
    }
    if (sorted)
        da_sort(table, n_tiles, [&](int i) {
            const Range r = da_blocks<true>(p, i / per_row, (i % per_row) * 128, 128);
            return r.end - r.begin;
        });
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_base_smem;

    struct Item {
        int b, t0, head;
        Range r;
        int n;
    };
    auto item_of = [&](int round, Item& m) {
        int tile;
        if (!da_item(round, n_tiles, p.heads, table, sorted, tile, m.head)) return false;
        m.b = tile / per_row;
        m.t0 = (tile % per_row) * 128;
        m.r = da_blocks<true>(p, m.b, m.t0, 128);
        m.n = m.r.end - m.r.begin;
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
                    const int s = it % S::STAGES, y = row + (m.r.begin + n) * 128;
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
        if (lane == 0) {
            bool ok = true;
            const uint32_t q_addr = smem_u32(sQ), do_addr = smem_u32(sDO);
            uint32_t it0 = 0, items = 0;
            Item m;
            for (int round = 0; ok && item_of(round, m); round++) {
                if (m.n == 0) continue;
                ok = mbar_wait(q_full, items & 1);
                for (int n = 0; n <= m.n && ok; n++) {
                    if (n < m.n) {
                        const uint32_t i = it0 + n;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&k_full[s], (i / S::STAGES) & 1);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint32_t k_addr = smem_u32(sK + s * S::TILE), v_addr = smem_u32(sV + s * S::TILE);
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {     // S = Q K^T : [128 queries x 128 keys]
                            const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                            umma_f16_ss(tmem_base + sb * 128, make_smem_desc_sw128(q_addr + off, 16, 1024), make_smem_desc_sw128(k_addr + off, 16, 1024), IDESC_S,
                                        kk != 0 ? 1u : 0u);
                        }
                        umma_commit(&s_full[sb]);
                        ok = mbar_wait(&v_full[s], (i / S::STAGES) & 1) && mbar_wait(dp_empty, (i & 1) ^ 1);
                        if (!ok) break;
                        tcgen05_fence_after();
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {     // dP = dO V^T
                            const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                            umma_f16_ss(tmem_base + 256, make_smem_desc_sw128(do_addr + off, 16, 1024), make_smem_desc_sw128(v_addr + off, 16, 1024), IDESC_S,
                                        kk != 0 ? 1u : 0u);
                        }
                        umma_commit(dp_full);
                        umma_commit(&v_empty[s]);
                        if (n == m.n - 1) umma_commit(q_empty);
                    }
                    if (n >= 1) {
                        const uint32_t i = it0 + n - 1;
                        const int sb = i & 1, s = i % S::STAGES;
                        ok = mbar_wait(&ds_full[sb], (i >> 1) & 1);
                        if (ok && n == 1) ok = mbar_wait(acc_empty, (items & 1) ^ 1);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint32_t k_addr = smem_u32(sK + s * S::TILE);
#pragma unroll
                        for (int kk = 0; kk < 8; kk++)            // dQ += dS K : dS [128 q x 128 keys] in tensor memory, K [128 keys x d], d contiguous
                            umma_f16_ts(tmem_base + 384, tmem_base + sb * 128 + (kk >> 2) * 64 + (kk & 3) * 8, make_smem_desc_sw128(k_addr + kk * 2048, 16384, 1024),
                                        IDESC_DQ, (n != 1 || kk != 0) ? 1u : 0u);
                        umma_commit(&k_empty[s]);
                    }
                }
                if (ok) umma_commit(acc_full);
                it0 += m.n;
                items++;
            }
            if (!ok) atomicExch(&g_doc_error, 22);
        }
    } else {
        // ---------------- row owners: two threads per query, 64 of the 128 key columns each ----------------
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int r = quarter * 32 + lane, c0 = half * 64;
        const uint32_t tm = tmem_base + ((uint32_t)(quarter * 32) << 16);
        bool ok = true;
        uint32_t it0 = 0, items = 0;
        Item m;
        for (int round = 0; item_of(round, m); round++) {
            const int qi = m.t0 + r;
            const bool live = qi < p.tokens;
            const int64_t row = (int64_t)m.b * p.tokens + qi;
            __half* dqrow = p.dq + row * p.ld_dq + m.head * D;
            if (m.n == 0) {
                if (half == 0 && live) da_zero_row(dqrow, D);
                continue;
            }
            int4 span = make_int4(0, 0x7fffffff, 0, 0);
            float lse2 = 0.0f, dlt = 0.0f;
            if (live) {
                const int64_t at = ((int64_t)m.b * p.heads + m.head) * p.tokens + qi;
                span = p.spans[row];
                lse2 = p.lse_in[at] * LOG2E;
                dlt = p.delta[at];
            }
            const int lo = max(span.x, 0), hi = live ? min(span.y, p.tokens) : span.y;
            const float slope2 = BIAS ? p.slopes[m.head] * LOG2E : 0.0f;
            const bool ahead = BIAS && __any_sync(0xffffffffu, live && hi > qi + 1);
            for (int n = 0; n < m.n && ok; n++) {
                const uint32_t i = it0 + n;
                const int sb = i & 1, kbase = (m.r.begin + n) * 128 + c0;
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[sb], (i >> 1) & 1) && mbar_wait(dp_full, i & 1));
                if (!ok) break;
                tcgen05_fence_after();
                const bool full = __all_sync(0xffffffffu, lo <= kbase && hi >= kbase + 64);
                const bool past = !ahead || __all_sync(0xffffffffu, kbase + 63 <= qi);
                const float dist = (float)(kbase - qi), base = fmaf(slope2, dist, -lse2);
                uint32_t w[2][16];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t sv[32], dv[32];
                    tmem_ld_32x32b_x32(tm + sb * 128 + c0 + c * 32, sv);
                    tmem_ld_32x32b_x32(tm + 256 + c0 + c * 32, dv);
                    tmem_ld_wait();
                    if (c == 1) {
                        tcgen05_fence_before();
                        mbar_arrive(dp_empty);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float de[2];
#pragma unroll
                        for (int f = 0; f < 2; f++) {
                            const int k = c * 32 + e + f;
                            float dt;
                            float s = da_score<CAP>(__uint_as_float(sv[e + f]), p, dt);
                            if (BIAS)
                                s += past ? fmaf(slope2, (float)k, base) : fmaf(-slope2, fabsf(dist + (float)k), -lse2);
                            else
                                s -= lse2;
                            de[f] = fast_exp2(s) * (__uint_as_float(dv[e + f]) - dlt);
                            if (CAP) de[f] *= dt;
                            if (!full && !(kbase + k >= lo && kbase + k < hi)) de[f] = 0.0f;
                        }
                        w[c][e >> 1] = da_half2(de[0], de[1]);
                    }
                }
                tmem_st_32x32b_x16(tm + sb * 128 + c0, w[0]);
                tmem_st_32x32b_x16(tm + sb * 128 + c0 + 16, w[1]);
                tmem_st_wait();
                tcgen05_fence_before();
                mbar_arrive(&ds_full[sb]);
            }
            it0 += m.n;
            if (ok) ok = mbar_wait(acc_full, items & 1);
            ok = __all_sync(0xffffffffu, ok);
            items++;
            const bool none = lo >= hi;
            float bad = 0.0f;
            if (ok) {
                tcgen05_fence_after();
#pragma unroll 1
                for (int d0 = half * (D / 2); d0 < (half + 1) * (D / 2); d0 += 32) {
                    uint32_t a[32];
                    tmem_ld_32x32b_x32(tm + 384 + d0, a);
                    tmem_ld_wait();
                    if (live) {
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            Vec<__half> o;
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const float x = __uint_as_float(a[g * 8 + e]);
                                bad = fmaf(x, 0.0f, bad);
                                o.v[e] = none ? 0.0f : x * p.scale;
                            }
                            o.store(dqrow + d0 + g * 8);
                        }
                    }
                }
                tcgen05_fence_before();
                mbar_arrive(acc_empty);
            }
            // evaluated again by the row's first owner, after both owners' stores (the barrier orders them)
            again[half * 128 + r] = bad;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (half == 0 && live && !none && (again[r] != 0.0f || again[128 + r] != 0.0f)) da_dq_row<D, CAP>(p, m.b, m.head, qi, lo, hi);
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (!ok && lane == 0) atomicExch(&g_doc_error, 23);
    }
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
static unsigned da_grid(int64_t items) { return (unsigned)(items < sm_count() ? items : sm_count()); }       // persistent: one CTA per SM walks the items

struct DocMaps {
    CUtensorMap q, k, v, d_out, q64, do64;
};

template <int D, bool CAP, bool BIAS>
static int da_fwd(const DocMaps& t, const DocAttn& p, cudaStream_t st) {
    constexpr size_t smem = FwdSmem<D>::BYTES;
    static_assert(smem <= 232448, "the tile set must fit the 227 KB a CTA can have");
    static std::atomic<uint64_t> done{0};
    const int rc = da_allow_smem(doc_attn_fwd_kernel<D, CAP, BIAS>, smem, done, "doc_attn_fwd smem attribute");
    if (rc) return rc;
    doc_attn_fwd_kernel<D, CAP, BIAS><<<da_grid((int64_t)p.batch * ((p.tokens + 255) / 256) * p.heads), DA_THREADS, smem, st>>>(t.q, t.k, t.v, p);
    return launch_status("doc_attn_fwd_kernel");
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
    doc_attn_dkv_kernel<D, CAP, BIAS><<<da_grid(tiles * p.kv_heads), DA_THREADS, smem_kv, st>>>(t.q64, t.k, t.v, t.do64, p);
    rc = launch_status("doc_attn_dkv_kernel");
    if (rc) return rc;
    doc_attn_dq_kernel<D, CAP, BIAS><<<da_grid(tiles * p.heads), DA_THREADS, smem_q, st>>>(t.q, t.k, t.v, t.d_out, p);
    return launch_status("doc_attn_dq_kernel");
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

// sizes, strides and alignment that both directions share
static int da_check(const void* q, const void* k, const void* v, int64_t ld_q, int64_t ld_kv, const void* out, int64_t ld_out, const int32_t* spans, float cap,
                    int batch, int tokens, int heads, int kv_heads, int d) {
    if (batch < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || (d != 64 && d != 128)) return BRK_ATTR_ERROR;
    if (heads > 4096 || tokens > (1 << 22) || (int64_t)batch * tokens > (1 << 30)) return BRK_ATTR_ERROR;
    if (!(cap >= 0.0f) || cap > 1e4f) return BRK_ATTR_ERROR;
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
    p.cap_in = cap > 0.0f ? (float)(2.0 * scale * log2e / cap) : 0.0f;
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
        !make_tmap_2d_f16(&t.v, v, rows, kc, (uint64_t)ld_kv, 64, 128)) {
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
        !make_tmap_2d_f16(&t.q64, q, rows, qc, (uint64_t)ld_q, 64, DA_SUB) || !make_tmap_2d_f16(&t.do64, d_out, rows, qc, (uint64_t)ld_out, 64, DA_SUB)) {
        set_error_message("brk_doc_attn_bwd: could not encode a tensor map");
        return BRK_CUDA_ERROR;
    }
    const int64_t threads = (int64_t)batch * tokens * heads * (head_dim / 8);
    doc_delta_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>((const __half*)out, (const __half*)d_out, ld_out, (float*)workspace, batch, tokens, heads,
                                                                       head_dim);
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
