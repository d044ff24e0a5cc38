// Spans and loss targets of packed documents.
//
// Rows of the batch hold several documents one after another, given as a number per token (0 or less = padding); a run
// of equal numbers is one document.  For every token the kernel finds where its run starts and ends and where the run's
// prompt ends (the first token of the run that is not marked as prompt), which are three scans over the tokens:
//     start = last run border at or before the token                       (running maximum from the left)
//     end   = first run border after it                                    (running minimum from the right)
//     pe    = first unmarked token at or after `start`, at most `end`      (running minimum from the right, taken at `start`)
// All rows are scanned as one sequence, since the first token of a row is a border.  One cluster of eight CTAs does it in
// one launch: a thread walks a strip of neighbouring tokens, strips meet by warp shuffles and shared memory, the CTAs'
// totals through distributed shared memory.  The work is latency (12 bytes in and 20 bytes out per token): 2 x 1024 tokens
// take 4.7 us, 8 x 8192 take 15.4 us, 136 GB/s.  More CTAs would have to meet through global memory, in a second launch.
#include "brk_common.cuh"
#include "brk_ptx.cuh"

namespace brk {

constexpr int DP_CTAS = 8;
constexpr int DP_NONE = 0x7fffffff;
constexpr int DP_NO_TARGET = -100;

struct DocPlanParams {
    const int32_t* mask;
    const int32_t* prompt;      // or null
    const int32_t* ids;         // or null
    int4* spans;
    int32_t* target;            // or null
    int32_t* count;             // or null
    int n, tokens, strip;       // n = batch * tokens
    bool wide;                  // 16-byte aligned inputs and targets
};

// address of this CTA's shared variable in CTA `rank` of the cluster, and loads from there
__device__ __forceinline__ uint32_t in_cta(const void* p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ int load_cta_i32(const int* p, int rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(in_cta(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long load_cta_u64(const unsigned long long* p, int rank) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(in_cta(p, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    ptx::cluster_sync_all();
}

__device__ __forceinline__ int2 min2(int2 a, int2 b) { return make_int2(min(a.x, b.x), min(a.y, b.y)); }
__device__ __forceinline__ unsigned long long max64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

struct DocPlanShared {
    int2 first[32];                                  // per warp: first border, first unmarked token
    unsigned long long last[32];                     // per warp: last border + 1 << 32 | its prompt's end
    int count[32];
    int2 all_first;                                  // this CTA's totals, read by the others
    unsigned long long all_last;
    int all_count;
};

// `own` of every strip to the strips before it: the least border and unmarked token behind this strip
__device__ __forceinline__ int2 plan_behind(int2 own, DocPlanShared& sh, int rank) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int2 suffix = own;                               // inclusive over the warp's lanes from the right
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int2 v = make_int2(__shfl_down_sync(0xffffffffu, suffix.x, o), __shfl_down_sync(0xffffffffu, suffix.y, o));
        if (lane + o < 32) suffix = min2(suffix, v);
    }
    if (lane == 0) sh.first[warp] = suffix;
    int2 after = make_int2(__shfl_down_sync(0xffffffffu, suffix.x, 1), __shfl_down_sync(0xffffffffu, suffix.y, 1));
    if (lane == 31) after = make_int2(DP_NONE, DP_NONE);
    __syncthreads();
    // the warps' values: one per lane, again a suffix minimum
    int2 w = lane < warps ? sh.first[lane] : make_int2(DP_NONE, DP_NONE);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int2 v = make_int2(__shfl_down_sync(0xffffffffu, w.x, o), __shfl_down_sync(0xffffffffu, w.y, o));
        if (lane + o < 32) w = min2(w, v);
    }
    if (threadIdx.x == 0) sh.all_first = w;
    const int2 next = make_int2(__shfl_sync(0xffffffffu, w.x, (warp + 1) & 31), __shfl_sync(0xffffffffu, w.y, (warp + 1) & 31));
    if (warp < 31) after = min2(after, next);
    cluster_meet();
    for (int r = rank + 1; r < DP_CTAS; r++) after = min2(after, make_int2(load_cta_i32(&sh.all_first.x, r), load_cta_i32(&sh.all_first.y, r)));
    return after;
}
// `own` of every strip to the strips behind it: the last border before this strip, with its prompt's end
__device__ __forceinline__ unsigned long long plan_before(unsigned long long own, DocPlanShared& sh, int rank) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    unsigned long long prefix = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, prefix, o);
        if (lane >= o) prefix = max64(prefix, v);
    }
    if (lane == 31) sh.last[warp] = prefix;
    unsigned long long before = __shfl_up_sync(0xffffffffu, prefix, 1);
    if (lane == 0) before = 0;
    __syncthreads();
    unsigned long long w = lane < warps ? sh.last[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w = max64(w, v);
    }
    if (threadIdx.x == 31) sh.all_last = w;
    const unsigned long long earlier = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    if (warp > 0) before = max64(before, earlier);
    cluster_meet();
    for (int r = 0; r < rank; r++) before = max64(before, load_cta_u64(&sh.all_last, r));
    return before;
}
__device__ __forceinline__ void plan_count(int counted, DocPlanShared& sh, int rank, int32_t* count) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    counted = __reduce_add_sync(0xffffffffu, counted);
    if (lane == 0) sh.count[warp] = counted;
    __syncthreads();
    if (warp == 0) {
        const int sum = __reduce_add_sync(0xffffffffu, lane < warps ? sh.count[lane] : 0);
        if (lane == 0) sh.all_count = sum;
    }
    cluster_meet();
    if (rank == 0 && threadIdx.x == 0) {
        int sum = 0;
        for (int r = 0; r < DP_CTAS; r++) sum += load_cta_i32(&sh.all_count, r);
        count[0] = sum;
    }
}

// A strip of S tokens that stays in registers: up to 65536 tokens in all.  8 x 8192 tokens: 44 us with the walk below, whose
// loads wait for one another.
template <int S>
__global__ void __cluster_dims__(DP_CTAS, 1, 1) __launch_bounds__(1024)
doc_plan_kernel(DocPlanParams p) {
    __shared__ DocPlanShared sh;
    const int rank = (int)ptx::cluster_ctarank();
    const int f0 = min((rank * (int)blockDim.x + (int)threadIdx.x) * S, p.n);
    int num[S + 2], id[S];                           // document numbers of the strip and of the tokens around it
    uint32_t marked = 0;                             // bit i: token f0 + i belongs to a prompt; bit S: the one behind the strip
    num[0] = f0 > 0 ? max(p.mask[f0 - 1], 0) : -1;
    if (S >= 4 && p.wide && f0 + S < p.n) {          // whole packets; the strips at the end take their tokens one by one
        alignas(16) int raw[S + 1];
        auto read = [&](const int32_t* from) {
#pragma unroll
            for (int i = 0; i < S; i += 4) *reinterpret_cast<int4*>(raw + i) = *reinterpret_cast<const int4*>(from + f0 + i);
            raw[S] = from[f0 + S];
        };
        read(p.mask);
#pragma unroll
        for (int i = 0; i <= S; i++) num[i + 1] = max(raw[i], 0);
        if (p.prompt) {
            read(p.prompt);
#pragma unroll
            for (int i = 0; i <= S; i++) marked |= (raw[i] != 0 ? 1u : 0u) << i;
        }
        if (p.target) {
            read(p.ids);
#pragma unroll
            for (int i = 0; i < S; i++) id[i] = raw[i + 1];
        }
    } else {
#pragma unroll
        for (int i = 0; i <= S; i++) {
            num[i + 1] = f0 + i < p.n ? max(p.mask[f0 + i], 0) : -1;
            if (p.prompt && f0 + i < p.n && p.prompt[f0 + i] != 0) marked |= 1u << i;
            if (i < S) id[i] = p.target && f0 + i + 1 < p.n ? p.ids[f0 + i + 1] : 0;
        }
    }
    const int t0 = f0 % p.tokens;
    uint32_t borders = 0;
    int column = t0;
#pragma unroll
    for (int i = 0; i < S; i++) {
        if (f0 + i < p.n && (column == 0 || num[i + 1] != num[i])) borders |= 1u << i;
        if (++column == p.tokens) column = 0;
    }
    const uint32_t here = f0 + S <= p.n ? (1u << S) - 1 : (1u << (p.n - f0)) - 1, open = ~marked & here;
    const int2 after = plan_behind(make_int2(borders ? f0 + __ffs(borders) - 1 : DP_NONE, open ? f0 + __ffs(open) - 1 : DP_NONE), sh, rank);
    int ends[S], answers[S];                         // end of the token's run; first unmarked token at or after it
    int e = min(after.x, p.n), a = min(after.y, p.n);
    unsigned long long last = 0;
#pragma unroll
    for (int i = S - 1; i >= 0; i--) {
        if (open >> i & 1) a = f0 + i;
        ends[i] = e;
        answers[i] = a;
        if (borders >> i & 1) {
            if (last == 0) last = (unsigned long long)(f0 + i + 1) << 32 | (unsigned)min(a, e);      // + 1: 0 means none
            e = f0 + i;
        }
    }
    const unsigned long long before = plan_before(last, sh, rank);
    int start = (int)(before >> 32) - 1, pe = (int)(before & 0xffffffffu), counted = 0, t = t0, aims[S];
#pragma unroll
    for (int i = 0; i < S; i++) {
        const int f = f0 + i;
        if (borders >> i & 1) {
            start = f;
            pe = min(answers[i], ends[i]);
        }
        if (f < p.n) {
            const int base = f - t, st = start - base, end = ends[i] - base, prompt_end = p.prompt ? pe - base : st;
            p.spans[f] = num[i + 1] > 0 ? make_int4(st, max(t + 1, prompt_end), t < prompt_end ? st : t, end) : make_int4(st, st, st, st);
            if (p.target) {
                const bool has = num[i + 1] > 0 && t + 1 < p.tokens && num[i + 2] == num[i + 1] && !(marked >> (i + 1) & 1);
                aims[i] = has ? id[i] : DP_NO_TARGET;
                counted += has;
            }
        }
        if (++t == p.tokens) t = 0;
    }
    if (p.target) {
        if (S >= 4 && p.wide && f0 + S <= p.n) {
#pragma unroll
            for (int i = 0; i < S; i += 4) *reinterpret_cast<int4*>(p.target + f0 + i) = make_int4(aims[i], aims[i + 1], aims[i + 2], aims[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < S; i++)
                if (f0 + i < p.n) p.target[f0 + i] = aims[i];
        }
    }
    if (p.count) plan_count(counted, sh, rank, p.count);
    cluster_meet();                                  // nobody leaves while its totals may still be read
}

// Strips of any length, walked three times.
__global__ void __cluster_dims__(DP_CTAS, 1, 1) __launch_bounds__(1024)
doc_plan_walk_kernel(DocPlanParams p) {
    __shared__ DocPlanShared sh;
    const int rank = (int)ptx::cluster_ctarank();
    const int64_t first = ((int64_t)rank * blockDim.x + threadIdx.x) * p.strip;
    const int f0 = (int)min(first, (int64_t)p.n), f1 = (int)min(first + p.strip, (int64_t)p.n);
    auto number = [&](int f) { return max(p.mask[f], 0); };
    auto border = [&](int f) { return f % p.tokens == 0 || number(f) != number(f - 1); };
    auto marked = [&](int f) { return p.prompt && p.prompt[f] != 0; };
    int2 own = make_int2(DP_NONE, DP_NONE);
    for (int f = f1 - 1; f >= f0; f--) {
        if (border(f)) own.x = f;
        if (!marked(f)) own.y = f;
    }
    const int2 after = plan_behind(own, sh, rank);
    // right to left: end of the run and first unmarked token at or after, kept in the output for the way back
    unsigned long long last = 0;
    int e = min(after.x, p.n), a = min(after.y, p.n);
    for (int f = f1 - 1; f >= f0; f--) {
        if (!marked(f)) a = f;
        p.spans[f] = make_int4(a, e, 0, 0);
        if (border(f)) {
            if (last == 0) last = (unsigned long long)(f + 1) << 32 | (unsigned)min(a, e);
            e = f;
        }
    }
    const unsigned long long before = plan_before(last, sh, rank);
    int start = (int)(before >> 32) - 1, pe = (int)(before & 0xffffffffu), counted = 0;
    for (int f = f0; f < f1; f++) {
        const int4 s = p.spans[f];
        if (border(f)) {
            start = f;
            pe = min(s.x, s.y);
        }
        const int num = number(f), base = f - f % p.tokens, t = f - base, st = start - base, end = s.y - base;
        const int prompt_end = p.prompt ? pe - base : st;
        p.spans[f] = num > 0 ? make_int4(st, max(t + 1, prompt_end), t < prompt_end ? st : t, end) : make_int4(st, st, st, st);
        if (p.target) {
            const bool has = num > 0 && t + 1 < p.tokens && number(f + 1) == num && !marked(f + 1);
            p.target[f] = has ? p.ids[f + 1] : DP_NO_TARGET;
            counted += has;
        }
    }
    if (p.count) plan_count(counted, sh, rank, p.count);
    cluster_meet();
}

}  // namespace brk

extern "C" int brk_doc_plan(const int32_t* mask, const int32_t* prompt, const int32_t* ids, int batch, int tokens, int32_t* spans, int32_t* target,
                            int32_t* count, void* stream) {
    using namespace brk;
    if (batch < 0 || tokens < 0 || (int64_t)batch * tokens > (1 << 30)) return BRK_ATTR_ERROR;
    if (count && !target && batch * tokens > 0) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    const int n = batch * tokens;
    if (n == 0) {
        if (!count) return BRK_OK;
        const cudaError_t e = cudaMemsetAsync(count, 0, sizeof(int32_t), st);
        if (e != cudaSuccess) {
            set_cuda_error(e, "doc_plan clear");
            return BRK_CUDA_ERROR;
        }
        return BRK_OK;
    }
    if (!mask || (target && !ids)) return BRK_INPUT_ERROR;
    if (!spans) return BRK_OUTPUT_ERROR;
    if (!aligned16(spans)) return BRK_ATTR_ERROR;
    DocPlanParams p = {mask, prompt, ids, (int4*)spans, target, count, n, tokens, 1, aligned16(mask) && aligned16(prompt) && aligned16(ids) && aligned16(target)};
    // few threads a CTA while a strip is short, then strips of up to eight tokens
    const int per_cta = (n + DP_CTAS - 1) / DP_CTAS;
    auto threads = [&](int strip) { return ((per_cta + strip - 1) / strip + 31) / 32 * 32; };
    if (per_cta <= 1024) doc_plan_kernel<1><<<DP_CTAS, threads(1), 0, st>>>(p);
    else if (per_cta <= 2048) doc_plan_kernel<2><<<DP_CTAS, threads(2), 0, st>>>(p);
    else if (per_cta <= 4096) doc_plan_kernel<4><<<DP_CTAS, threads(4), 0, st>>>(p);
    else if (per_cta <= 8192) doc_plan_kernel<8><<<DP_CTAS, threads(8), 0, st>>>(p);
    else {
        p.strip = (per_cta + 1023) / 1024;
        doc_plan_walk_kernel<<<DP_CTAS, 1024, 0, st>>>(p);
    }
    return launch_status("doc_plan_kernel");
}
