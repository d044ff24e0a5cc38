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
// totals through distributed shared memory.  The work is latency: 12 bytes in and 20 bytes out per token.
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

__global__ void __cluster_dims__(DP_CTAS, 1, 1) __launch_bounds__(1024)
doc_plan_kernel(DocPlanParams p) {
    const int rank = (int)ptx::cluster_ctarank();
    __shared__ int2 s_min[32];                       // per warp: first border, first unmarked token
    __shared__ unsigned long long s_max[32];         // per warp: last border << 32 | its prompt's end
    __shared__ int s_count[32];
    __shared__ int2 t_min;                           // this CTA's totals, read by the others
    __shared__ unsigned long long t_max;
    __shared__ int t_count;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t first = ((int64_t)rank * blockDim.x + threadIdx.x) * p.strip;
    const int f0 = (int)min(first, (int64_t)p.n), f1 = (int)min(first + p.strip, (int64_t)p.n);
    auto number = [&](int f) { return max(p.mask[f], 0); };
    auto border = [&](int f) { return f % p.tokens == 0 || number(f) != number(f - 1); };
    auto marked = [&](int f) { return p.prompt && p.prompt[f] != 0; };

    // from the right: what this strip offers to the ones before it
    int2 own = make_int2(DP_NONE, DP_NONE);
    for (int f = f1 - 1; f >= f0; f--) {
        if (border(f)) own.x = f;
        if (!marked(f)) own.y = f;
    }
    int2 suffix = own;                               // inclusive over the warp's lanes from the right
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int2 v = make_int2(__shfl_down_sync(0xffffffffu, suffix.x, o), __shfl_down_sync(0xffffffffu, suffix.y, o));
        if (lane + o < 32) suffix = min2(suffix, v);
    }
    if (lane == 0) s_min[warp] = suffix;
    int2 after = make_int2(__shfl_down_sync(0xffffffffu, suffix.x, 1), __shfl_down_sync(0xffffffffu, suffix.y, 1));
    if (lane == 31) after = make_int2(DP_NONE, DP_NONE);
    __syncthreads();
    int2 total = make_int2(DP_NONE, DP_NONE);
    for (int w = warps - 1; w >= 0; w--) {
        if (w > warp) after = min2(after, s_min[w]);
        total = min2(total, s_min[w]);
    }
    if (threadIdx.x == 0) t_min = total;
    cluster_meet();
    for (int r = rank + 1; r < DP_CTAS; r++) after = min2(after, make_int2(load_cta_i32(&t_min.x, r), load_cta_i32(&t_min.y, r)));

    // right to left through the strip: end of the run and first unmarked token at or after; kept in the output for the
    // walk back.  The strip's last border goes on to the strips after it.
    unsigned long long last = 0;
    {
        int e = min(after.x, p.n), a = min(after.y, p.n);
        for (int f = f1 - 1; f >= f0; f--) {
            if (!marked(f)) a = f;
            p.spans[f] = make_int4(a, e, 0, 0);
            if (border(f)) {
                if (last == 0) last = (unsigned long long)(f + 1) << 32 | (unsigned)min(a, e);      // f + 1: 0 means none
                e = f;
            }
        }
    }
    unsigned long long prefix = last;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, prefix, o);
        if (lane >= o) prefix = max64(prefix, v);
    }
    if (lane == 31) s_max[warp] = prefix;
    unsigned long long before = __shfl_up_sync(0xffffffffu, prefix, 1);
    if (lane == 0) before = 0;
    __syncthreads();
    unsigned long long top = 0;
    for (int w = 0; w < warps; w++) {
        if (w < warp) before = max64(before, s_max[w]);
        top = max64(top, s_max[w]);
    }
    if (threadIdx.x == 0) t_max = top;
    cluster_meet();
    for (int r = 0; r < rank; r++) before = max64(before, load_cta_u64(&t_max, r));

    // left to right: the spans, relative to the token's row, and the targets
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
    if (p.count) {
        counted = __reduce_add_sync(0xffffffffu, counted);
        if (lane == 0) s_count[warp] = counted;
        __syncthreads();
        if (warp == 0) {
            const int sum = __reduce_add_sync(0xffffffffu, lane < warps ? s_count[lane] : 0);
            if (lane == 0) t_count = sum;
        }
        cluster_meet();
        if (rank == 0 && threadIdx.x == 0) {
            int sum = 0;
            for (int r = 0; r < DP_CTAS; r++) sum += load_cta_i32(&t_count, r);
            p.count[0] = sum;
        }
    }
    cluster_meet();                                  // nobody leaves while its totals may still be read
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
    DocPlanParams p = {mask, prompt, ids, (int4*)spans, target, count, n, tokens, 1};
    const int per_cta = (n + DP_CTAS - 1) / DP_CTAS;
    const int threads = per_cta >= 1024 ? 1024 : (per_cta + 31) / 32 * 32;
    p.strip = (per_cta + threads - 1) / threads;
    doc_plan_kernel<<<DP_CTAS, threads, 0, st>>>(p);
    return launch_status("doc_plan_kernel");
}
