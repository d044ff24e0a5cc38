// Activations kept in 8 bits between the forward and the backward pass.
//
// A row is cut into blocks of 128 columns (the last one may be shorter).  With top = the largest magnitude of a block
//     q = rint(x * 127 / top)   (int8),     scale = top / 127   (fp32),     the kept value is q * scale,
// so a kept value is off by at most half a step, top / 254, of its own block: an outlier column coarsens its 127
// neighbours in that row and nothing else.  int8 and not an 8-bit float: inside a block of normalised activations the
// magnitudes span two or three powers of two, and there the uniform step of 1/127 of the largest is finer than the
// 2^-4 of the value itself that a float with three mantissa bits leaves.  A block that holds an infinity or a NaN gets
// the scale NaN, so every value of it reads NaN: an overflow stays visible.  A block whose largest magnitude is below
// 2^-119 (where 127 / top would overflow) is kept as zeros.
//
// LayerNorm keeps the normalised row xhat and not y = xhat * gamma + beta: xhat = (y - beta) / gamma would divide the
// rounding error by gamma.
//
// All of it is bound by HBM: one pass, 16-byte accesses, everything that a block shares travels by warp shuffles.  fp16:
// GELU of [8192, 16384] 119 us forward and 162 us backward, 5.7 and 5.8 TB/s (gelu(x) written again with dx); LayerNorm of
// [8192, 4096] 35 us and 62 us; [2048, 4096] packed in 6.3 us, unpacked in 5.4 us.
#include <mutex>

#include "brk_common.cuh"

namespace brk {

constexpr int A8_BLOCK = 128;                 // columns that share a scale
constexpr int A8_THREADS = 256;
constexpr float A8_TINY = 1.5046328e-36f;     // 2^-119

// ---- 8-bit arithmetic ----------------------------------------------------------------------------------------------

// largest magnitude as a bit pattern: NaN and infinity order above every number
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// 127 / top, with EXACT in two parts, and the scale
struct A8Scale {
    float inv, rest, scale;
};
// EXACT: x * 127 / top correctly rounded, so that a value in the middle between two steps (half of the block's largest, say; a
// few fp16 values in ten thousand) stays there and goes to even as it does in exact arithmetic.  Normalised rows, in fp32,
// hold no such values, and a rounding of 2^-22 there saves 20 instructions a block.
template <bool EXACT = true>
__device__ __forceinline__ A8Scale a8_scale(uint32_t top_bits) {
    A8Scale s;
    const float top = __uint_as_float(top_bits);
    s.rest = 0.0f;
    if (top_bits >= 0x7f800000u) {
        s.inv = 0.0f;
        s.scale = __uint_as_float(0x7fffffffu);
    } else if (top < A8_TINY) {
        s.inv = 0.0f;
        s.scale = 0.0f;
    } else {
        s.inv = EXACT ? __fdiv_rn(127.0f, top) : __fdividef(127.0f, top);
        if (EXACT) s.rest = fmaf(-s.inv, top, 127.0f) * (s.inv * (1.0f / 127.0f));
        s.scale = top * (1.0f / 127.0f);
    }
    return s;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// Four values to four bytes.  Adding 1.5 * 2^23 leaves the nearest integer (ties to even) in the low mantissa bits, and
// a byte permute gathers them: no conversion instruction, which would run at an eighth of the rate.  With inv == 0 the product is
// 0, or NaN for a value that is not finite; its low byte is whatever it is, the block's scale is NaN then.
template <bool EXACT = true>
__device__ __forceinline__ float2 a8_step(float2 x, const A8Scale& s) {
    return EXACT ? __ffma2_rn(x, both(s.inv), __fmul2_rn(x, both(s.rest))) : __fmul2_rn(x, both(s.inv));
}
template <bool EXACT = true>
__device__ __forceinline__ uint32_t a8_pack4(float2 a, float2 b, const A8Scale& s) {
    const float2 x = __fadd2_rn(a8_step<EXACT>(a, s), both(12582912.0f)), y = __fadd2_rn(a8_step<EXACT>(b, s), both(12582912.0f));
    return __byte_perm(__byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040), __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040), 0x5410);
}
__device__ __forceinline__ int8_t a8_pack1(float x, const A8Scale& s) {
    return (int8_t)(__float_as_uint(__fadd_rn(fmaf(x, s.inv, __fmul_rn(x, s.rest)), 12582912.0f)) & 0xff);
}
__device__ __forceinline__ uint4 a8_pack16(const float2 (&v)[8], const A8Scale& s) {
    return make_uint4(a8_pack4(v[0], v[1], s), a8_pack4(v[2], v[3], s), a8_pack4(v[4], v[5], s), a8_pack4(v[6], v[7], s));
}
// Two bytes of a word as the numbers they stand for: 2^23 + (b + 128) assembled from its bits, exactly.
template <int B>
__device__ __forceinline__ float2 a8_bytes(uint32_t flipped) {
    const float2 f = make_float2(__uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7440 + B)), __uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7441 + B)));
    return __fadd2_rn(f, both(-8388736.0f));
}
__device__ __forceinline__ void a8_unpack16(const uint4& w, float scale, float2 (&o)[8]) {
    const uint32_t x[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        o[2 * i] = __fmul2_rn(a8_bytes<0>(x[i]), both(scale));
        o[2 * i + 1] = __fmul2_rn(a8_bytes<2>(x[i]), both(scale));
    }
}

// ---- 16 consecutive columns of storage type T, packed until used ------------------------------------------------------
template <typename T>
struct Pack16 {
    static constexpr int VN = Vec<T>::N, N = 16 / VN;
    uint4 v[N];
    __device__ __forceinline__ void stream(const T* p) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = ld_raw_stream(p + i * VN);
    }
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = ld_raw(p + i * VN);
    }
    __device__ __forceinline__ void to(float2 (&o)[8]) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            Vec<T> x;
            x.unpack(v[i]);
#pragma unroll
            for (int e = 0; e < VN; e += 2) o[(i * VN + e) / 2] = make_float2(x.v[e], x.v[e + 1]);
        }
    }
};
template <typename T>
__device__ __forceinline__ void store16(T* p, const float2 (&x)[8]) {
    constexpr int VN = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < 16 / VN; i++) {
        Vec<T> v;
#pragma unroll
        for (int e = 0; e < VN; e += 2) {
            v.v[e] = x[(i * VN + e) / 2].x;
            v.v[e + 1] = x[(i * VN + e) / 2].y;
        }
        v.store_stream(p + i * VN);
    }
}

// ---- bloom GELU in fp32: tanh(u) = 1 - 2 / (1 + exp(2u)), absolute error about 1e-7 -----------------------------------
struct GeluTerms {
    float y, dy;      // gelu(x) and its derivative
};
template <typename T>
__device__ __forceinline__ GeluTerms gelu_terms(float x) {
    const float x2 = x * x;
    const float t = 1.0f - __fdividef(2.0f, __expf(x * fmaf(2.0f * 0.79788456f * 0.044715f, x2, 2.0f * 0.79788456f)) + 1.0f);
    const float hx = 0.5f * x;
    GeluTerms r;
    r.y = fmaf(hx, t, hx);
    const float slope2 = sizeof(T) == 4 ? fminf(x2, 1e36f) : x2;      // finite where fp32 values overflow it: 1 - t^2 is 0 long before
    r.dy = fmaf(hx * fmaf(-t, t, 1.0f), fmaf(3.0f * 0.79788456f * 0.044715f, slope2, 0.79788456f), fmaf(0.5f, t, 0.5f));
    return r;
}

// ---- pack, and GELU that keeps its input: a thread owns 16 columns, 8 neighbouring lanes a block ----------------------
// units_per_row counts 16-column units with the last block filled up to 8 of them, so that a block never leaves its lanes.
// Two units of a thread are in flight at once.
constexpr int A8_UNITS = 2;
struct A8Unit {
    int64_t at;          // first element
    bool live;
};
__device__ __forceinline__ A8Unit a8_unit(int64_t u, int64_t units, int units_per_row, int cols, bool whole) {
    A8Unit r = {u * 16, u < units};
    if (!whole) {
        const int64_t row = u / units_per_row;
        const int c = (int)(u - row * units_per_row) * 16;
        r.live = r.live && c < cols;
        r.at = row * cols + c;
    }
    return r;
}
template <typename T, bool GELU>
__global__ void __launch_bounds__(A8_THREADS)
a8_pack_kernel(const T* x, T* y, int8_t* __restrict__ q, float* __restrict__ scale, int64_t units, int units_per_row, int cols) {
    pdl_wait();
    const bool whole = (cols & (A8_BLOCK - 1)) == 0;
    const int64_t stride = (int64_t)gridDim.x * A8_THREADS;
    for (int64_t u0 = (int64_t)blockIdx.x * A8_THREADS + threadIdx.x; u0 - threadIdx.x % 32 < units; u0 += A8_UNITS * stride) {
        A8Unit unit[A8_UNITS];
        Pack16<T> raw[A8_UNITS] = {};
#pragma unroll
        for (int i = 0; i < A8_UNITS; i++) {
            unit[i] = a8_unit(u0 + i * stride, units, units_per_row, cols, whole);
            if (unit[i].live) raw[i].stream(x + unit[i].at);
        }
#pragma unroll
        for (int i = 0; i < A8_UNITS; i++) {
            float2 v[8];
            raw[i].to(v);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, max(mag_bits(v[e].x), mag_bits(v[e].y)));
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (unit[i].live) {
                const A8Scale s = a8_scale(top);
                __stcs(reinterpret_cast<uint4*>(q + unit[i].at), a8_pack16(v, s));
                if ((threadIdx.x & 7) == 0) scale[(u0 + i * stride) >> 3] = s.scale;
                if (GELU) {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = make_float2(gelu_terms<T>(v[e].x).y, gelu_terms<T>(v[e].y).y);
                    store16(y + unit[i].at, v);
                }
            }
        }
    }
    pdl_launch_dependents();
}

// any column count and alignment: a warp owns a block, scalar accesses
template <typename T, bool GELU>
__global__ void __launch_bounds__(A8_THREADS)
a8_pack_generic_kernel(const T* x, T* y, int8_t* q, float* scale, int64_t rows, int blocks, int cols) {
    const int lane = threadIdx.x & 31;
    for (int64_t w = ((int64_t)blockIdx.x * A8_THREADS + threadIdx.x) >> 5; w < rows * blocks; w += ((int64_t)gridDim.x * A8_THREADS) >> 5) {
        const int64_t row = w / blocks;
        const int c0 = (int)(w - row * blocks) * A8_BLOCK;
        const int64_t at = row * cols + c0;
        float v[4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = i * 32 + lane;
            v[i] = c0 + c < cols ? to_f32(x[at + c]) : 0.0f;
            top = max(top, mag_bits(v[i]));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const A8Scale s = a8_scale(top);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = i * 32 + lane;
            if (c0 + c < cols) {
                q[at + c] = a8_pack1(v[i], s);
                if (GELU) y[at + c] = from_f32<T>(gelu_terms<T>(v[i]).y);
            }
        }
        if (lane == 0) scale[w] = s.scale;
    }
}

// ---- unpack (DY = false): out = q * scale.  GELU backward: dx = dy * gelu'(q * scale), and gelu(q * scale) again when y --
template <typename T, bool DY>
__global__ void __launch_bounds__(A8_THREADS)
a8_unpack_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, const T* dy, T* out, T* y, int64_t units, int units_per_row, int cols) {
    pdl_wait();
    const bool whole = (cols & (A8_BLOCK - 1)) == 0;
    const int64_t stride = (int64_t)gridDim.x * A8_THREADS;
    for (int64_t u0 = (int64_t)blockIdx.x * A8_THREADS + threadIdx.x; u0 < units; u0 += A8_UNITS * stride) {
        A8Unit unit[A8_UNITS];
        Pack16<T> g[A8_UNITS];
        uint4 w[A8_UNITS];
        float s[A8_UNITS];
#pragma unroll
        for (int i = 0; i < A8_UNITS; i++) {
            unit[i] = a8_unit(u0 + i * stride, units, units_per_row, cols, whole);
            if (unit[i].live) {
                w[i] = __ldcs(reinterpret_cast<const uint4*>(q + unit[i].at));
                s[i] = scale[(u0 + i * stride) >> 3];
                if (DY) g[i].stream(dy + unit[i].at);
            }
        }
#pragma unroll
        for (int i = 0; i < A8_UNITS; i++) {
            if (!unit[i].live) continue;
            float2 v[8];
            a8_unpack16(w[i], s[i], v);
            if (DY) {
                float2 d[8];
                g[i].to(d);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const GeluTerms t0 = gelu_terms<T>(v[e].x), t1 = gelu_terms<T>(v[e].y);
                    d[e] = __fmul2_rn(d[e], make_float2(t0.dy, t1.dy));
                    v[e] = make_float2(t0.y, t1.y);
                }
                store16(out + unit[i].at, d);
                if (y) store16(y + unit[i].at, v);
            } else {
                store16(out + unit[i].at, v);
            }
        }
    }
    pdl_launch_dependents();
}

template <typename T, bool DY>
__global__ void __launch_bounds__(A8_THREADS)
a8_unpack_generic_kernel(const int8_t* q, const float* scale, const T* dy, T* out, T* y, int64_t rows, int blocks, int cols) {
    const int lane = threadIdx.x & 31;
    for (int64_t w = ((int64_t)blockIdx.x * A8_THREADS + threadIdx.x) >> 5; w < rows * blocks; w += ((int64_t)gridDim.x * A8_THREADS) >> 5) {
        const int64_t row = w / blocks;
        const int c0 = (int)(w - row * blocks) * A8_BLOCK;
        const int64_t at = row * cols + c0;
        const float s = scale[w];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = i * 32 + lane;
            if (c0 + c < cols) {
                const float v = (float)q[at + c] * s;
                if (DY) {
                    const GeluTerms t = gelu_terms<T>(v);
                    out[at + c] = from_f32<T>(to_f32(dy[at + c]) * t.dy);
                    if (y) y[at + c] = from_f32<T>(t.y);
                } else {
                    out[at + c] = from_f32<T>(v);
                }
            }
        }
    }
}

static int a8_grid(int64_t threads) {
    const int64_t want = (threads + A8_THREADS - 1) / A8_THREADS, cap = (int64_t)sm_count() * 16;
    return (int)(want < cap ? want : cap);
}

template <typename T, bool GELU>
static int a8_pack(const void* x, void* y, int8_t* q, float* scale, int64_t rows, int64_t cols, cudaStream_t st) {
    const int blocks = (int)((cols + A8_BLOCK - 1) / A8_BLOCK);
    if (cols % 16 == 0 && aligned16(x) && aligned16(q) && (!GELU || aligned16(y))) {
        const int64_t units = rows * blocks * 8;
        const cudaError_t e = launch_pdl(a8_pack_kernel<T, GELU>, a8_grid(units), A8_THREADS, 0, st, (const T*)x, (T*)y, q, scale, units, blocks * 8, (int)cols);
        if (e != cudaSuccess) {
            set_cuda_error(e, "a8_pack_kernel");
            return BRK_CUDA_ERROR;
        }
        return launch_status("a8_pack_kernel");
    }
    a8_pack_generic_kernel<T, GELU><<<a8_grid(rows * blocks * 32), A8_THREADS, 0, st>>>((const T*)x, (T*)y, q, scale, rows, blocks, (int)cols);
    return launch_status("a8_pack_generic_kernel");
}

template <typename T, bool DY>
static int a8_unpack(const int8_t* q, const float* scale, const void* dy, void* out, void* y, int64_t rows, int64_t cols, cudaStream_t st) {
    const int blocks = (int)((cols + A8_BLOCK - 1) / A8_BLOCK);
    if (cols % 16 == 0 && aligned16(q) && aligned16(out) && (!DY || aligned16(dy)) && (!y || aligned16(y))) {
        const int64_t units = rows * blocks * 8;
        const cudaError_t e = launch_pdl(a8_unpack_kernel<T, DY>, a8_grid(units), A8_THREADS, 0, st, q, scale, (const T*)dy, (T*)out, (T*)y, units, blocks * 8, (int)cols);
        if (e != cudaSuccess) {
            set_cuda_error(e, "a8_unpack_kernel");
            return BRK_CUDA_ERROR;
        }
        return launch_status("a8_unpack_kernel");
    }
    a8_unpack_generic_kernel<T, DY><<<a8_grid(rows * blocks * 32), A8_THREADS, 0, st>>>(q, scale, (const T*)dy, (T*)out, (T*)y, rows, blocks, (int)cols);
    return launch_status("a8_unpack_generic_kernel");
}

// ---- LayerNorm ---------------------------------------------------------------------------------------------------------
// A thread owns groups of 8 columns, so 16 neighbouring lanes are a block of 128; a row (of up to 8192 columns) is owned by
// a team of `team` threads, a multiple of 32, thread t with the columns from 8 t, 8 (team + t) and so on, and a CTA
// holds blockDim.x / team teams that meet at named barriers of their own and never wait for one another.  Every thread copies
// its own packets of the next rows into slots of its own with cp.async, several rows ahead and without a barrier: the two
// reductions of a row leave the memory system idle otherwise, and registers hold one row ahead at most ([8192, 4096] fp16
// backward: 85 us with one row ahead in registers).
constexpr int A8_LN_MAX_COLS = 8192;
constexpr int A8_LN_THREADS = 512;

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(to);
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(a), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 8 columns of storage type T
template <typename T>
struct Group8 {
    static constexpr int N = 8 / Vec<T>::N;          // 16-byte packets
    // slot p of a stage lies at [p][thread]
    static __device__ __forceinline__ void fetch(uint4* slot, int threads, const T* from) {
#pragma unroll
        for (int i = 0; i < N; i++) copy_async<16>(slot + i * threads, from + i * Vec<T>::N);
    }
    static __device__ __forceinline__ void read(const uint4* slot, int threads, float2* o) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            Vec<T> x;
            x.unpack(slot[i * threads]);
#pragma unroll
            for (int e = 0; e < Vec<T>::N; e += 2) o[(i * Vec<T>::N + e) / 2] = make_float2(x.v[e], x.v[e + 1]);
        }
    }
    static __device__ __forceinline__ void write(T* to, const float2* x) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < Vec<T>::N; e += 2) {
                v.v[e] = x[(i * Vec<T>::N + e) / 2].x;
                v.v[e + 1] = x[(i * Vec<T>::N + e) / 2].y;
            }
            v.store_stream(to + i * Vec<T>::N);
        }
    }
    static __device__ __forceinline__ void load(const T* from, float2* o) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            Vec<T> x;
            x.load(from + i * Vec<T>::N);
#pragma unroll
            for (int e = 0; e < Vec<T>::N; e += 2) o[(i * Vec<T>::N + e) / 2] = make_float2(x.v[e], x.v[e + 1]);
        }
    }
};
__device__ __forceinline__ void a8_unpack8(const uint2& w, float scale, float2* o) {
    const uint32_t x[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        o[2 * i] = __fmul2_rn(a8_bytes<0>(x[i]), both(scale));
        o[2 * i + 1] = __fmul2_rn(a8_bytes<2>(x[i]), both(scale));
    }
}

__device__ __forceinline__ void team_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// Sums over the team; red: one cell per warp of the team, used alternately by the caller (two buffers) so that one barrier per
// reduction is enough.
__device__ __forceinline__ float team_sum(float a, float* red, int id, int team) {
    a = warp_sum(a);
    if (team == 32) return a;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x % team) >> 5, warps = team >> 5;
    if (lane == 0) red[warp] = a;
    team_barrier(id, team);
    return warp_sum(lane < warps ? red[lane] : 0.0f);
}
__device__ __forceinline__ float2 team_sum2(float a, float b, float2* red, int id, int team) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (team == 32) return make_float2(a, b);
    const int lane = threadIdx.x & 31, warp = (threadIdx.x % team) >> 5, warps = team >> 5;
    if (lane == 0) red[warp] = make_float2(a, b);
    team_barrier(id, team);
    const float2 t = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
    return make_float2(warp_sum(t.x), warp_sum(t.y));
}

// Forward: a thread owns four groups of 8 columns (8 (k * team + t) on), which halves what the reductions cost an element
// against two.  gamma and beta wait in shared memory, in fp32: unpacking them for every row took a quarter of the time.
template <typename T>
struct LnFwd {
    static constexpr int K = 4, STAGES = 4, THREADS = 256;
    static constexpr int CTAS = sizeof(T) == 2 ? 2 : 1;             // resident on an SM
    static constexpr size_t PER_THREAD = STAGES * K * 8 * sizeof(T), PER_MEMBER = 2 * K * 8 * sizeof(float);       // bytes of a thread; of a member of a team
};
template <typename T>
__global__ void __launch_bounds__(256, LnFwd<T>::CTAS)
a8_ln_fwd_kernel(const T* x, const T* __restrict__ gamma, const T* __restrict__ beta, T* y, int8_t* __restrict__ q,
                 float* __restrict__ scale, float* __restrict__ var, int64_t rows, int cols, float eps, int team) {
    using G = Group8<T>;
    constexpr int STAGES = LnFwd<T>::STAGES, K = LnFwd<T>::K, E = 4 * K;       // E: pairs of columns
    extern __shared__ __align__(16) unsigned char ln_smem[];
    __shared__ float red[2][LnFwd<T>::THREADS / 32];        // [buffer][warp of the CTA]: a team uses its own warps' cells
    const int threads = blockDim.x;
    const int tid = threadIdx.x % team, group = threadIdx.x / team, groups = threads / team;
    const int blocks = (cols + A8_BLOCK - 1) / A8_BLOCK;
    const int c0 = tid * 8, cstep = team * 8;
    const float inv_n = 1.0f / (float)cols;
    float* r0 = red[0] + group * (team >> 5);
    float* r1 = red[1] + group * (team >> 5);
    uint4* const slots = reinterpret_cast<uint4*>(ln_smem) + threadIdx.x;                          // [stage][group of columns][packet][thread]
    float2* const ga = reinterpret_cast<float2*>(ln_smem + (size_t)threads * LnFwd<T>::PER_THREAD) + tid;       // gamma [E][member], beta [E][member]
    float2* const be = ga + E * team;
    if (group == 0) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            float2 g[4] = {}, b[4] = {};
            if (c0 + k * cstep < cols) {
                G::load(gamma + c0 + k * cstep, g);
                G::load(beta + c0 + k * cstep, b);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                ga[(4 * k + e) * team] = g[e];
                be[(4 * k + e) * team] = b[e];
            }
        }
    }
    for (int i = 0; i < STAGES * K * G::N; i++)              // columns beyond the last stay zero
        if (c0 + (i / G::N) % K * cstep >= cols) slots[i * threads] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    pdl_wait();
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + group;
    auto fetch = [&](int64_t at, int stage) {
        if (at < rows) {
            const T* from = x + at * cols;
            uint4* slot = slots + stage * K * G::N * threads;
#pragma unroll
            for (int k = 0; k < K; k++)
                if (c0 + k * cstep < cols) G::fetch(slot + k * G::N * threads, threads, from + c0 + k * cstep);
        }
        copy_commit();
    };
    for (int i = 0; i < STAGES - 1; i++) fetch(row + i * step, i);
    for (int stage = 0; row < rows; row += step, stage = stage + 1 == STAGES ? 0 : stage + 1) {
        copy_wait<STAGES - 2>();
        fetch(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
        float2 v[E];
        const uint4* slot = slots + stage * K * G::N * threads;
#pragma unroll
        for (int k = 0; k < K; k++) G::read(slot + k * G::N * threads, threads, v + 4 * k);
        float2 s[2] = {v[0], v[1]};
#pragma unroll
        for (int e = 2; e < E; e++) s[e & 1] = __fadd2_rn(s[e & 1], v[e]);
        s[0] = __fadd2_rn(s[0], s[1]);
        const float mu = team_sum(s[0].x + s[0].y, r0, group + 1, team) * inv_n;
        float2 d2[2] = {both(0.0f), both(0.0f)};
#pragma unroll
        for (int e = 0; e < E; e++) {
            v[e] = __fadd2_rn(v[e], both(-mu));
            if (c0 + e / 4 * cstep < cols) d2[e & 1] = __ffma2_rn(v[e], v[e], d2[e & 1]);
        }
        d2[0] = __fadd2_rn(d2[0], d2[1]);
        const float va = fmaf(team_sum(d2[0].x + d2[0].y, r1, group + 1, team), inv_n, eps);
        const float rstd = rsqrtf(va);
        float top[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            top[k] = 0.0f;
#pragma unroll
            for (int e = 4 * k; e < 4 * k + 4; e++) {
                v[e] = __fmul2_rn(v[e], both(rstd));
                top[k] = max3(top[k], fabsf(v[e].x), fabsf(v[e].y));
            }
            if (c0 + k * cstep >= cols) top[k] = 0.0f;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < K; k++) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
        // a value that is not finite makes the row's variance so, and every normalised value with it
        const bool finite = va < INFINITY;
        const int64_t at = row * cols;
        int8_t* const qr = q + at;
        T* const yr = y + at;
        float* const sr = scale + row * blocks;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = c0 + k * cstep;
            if (c >= cols) continue;
            const A8Scale sc = a8_scale<false>(finite ? __float_as_uint(top[k]) : 0x7fffffffu);
            __stcs(reinterpret_cast<uint2*>(qr + c), make_uint2(a8_pack4<false>(v[4 * k], v[4 * k + 1], sc), a8_pack4<false>(v[4 * k + 2], v[4 * k + 3], sc)));
            if ((threadIdx.x & 15) == 0) sr[c >> 7] = sc.scale;
            float2 o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = __ffma2_rn(v[4 * k + e], ga[(4 * k + e) * team], be[(4 * k + e) * team]);
            G::write(yr + c, o);
        }
        if (tid == 0) var[row] = va;
    }
    copy_wait<0>();
    pdl_launch_dependents();
}

// any column count and alignment: one CTA per row, the row read three times
template <typename T>
__global__ void __launch_bounds__(A8_THREADS)
a8_ln_fwd_generic_kernel(const T* x, const T* gamma, const T* beta, T* y, int8_t* q, float* scale, float* var, int cols, float eps) {
    __shared__ float red[64];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * cols;
    const int blocks = (cols + A8_BLOCK - 1) / A8_BLOCK, lane = threadIdx.x & 31;
    float s = 0.0f, z = 0.0f;
    for (int i = threadIdx.x; i < cols; i += A8_THREADS) s += to_f32(xr[i]);
    block_sum2(s, z, red);
    const float mu = s / (float)cols;
    float d2 = 0.0f;
    z = 0.0f;
    for (int i = threadIdx.x; i < cols; i += A8_THREADS) {
        const float d = to_f32(xr[i]) - mu;
        d2 = fmaf(d, d, d2);
    }
    block_sum2(d2, z, red);
    const float va = d2 / (float)cols + eps, rstd = rsqrtf(va);
    for (int b = threadIdx.x >> 5; b < blocks; b += A8_THREADS / 32) {
        float v[4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = b * A8_BLOCK + i * 32 + lane;
            v[i] = c < cols ? (to_f32(xr[c]) - mu) * rstd : 0.0f;
            top = max(top, mag_bits(v[i]));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const A8Scale sc = a8_scale(top);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = b * A8_BLOCK + i * 32 + lane;
            if (c < cols) {
                q[row * cols + c] = a8_pack1(v[i], sc);
                y[row * cols + c] = from_f32<T>(fmaf(v[i], to_f32(gamma[c]), to_f32(beta[c])));
            }
        }
        if (lane == 0) scale[row * blocks + b] = sc.scale;
    }
    if (threadIdx.x == 0) var[row] = va;
}

// Backward.  g = dy * gamma;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) (+ residual);  the column sums of
// dy * xhat and dy stay in the registers of the column's owner over all rows of the CTA, are added over the CTA's teams
// through shared memory and leave as one row of `part` [gridDim.x][2][cols], which a second kernel adds in order.
// What is needed on both sides of the barrier is unpacked twice rather than held in 32 bits, which would not fit the registers.
template <typename T, bool RES>
struct LnBwdSmem {
    static constexpr int STAGES = sizeof(T) == 2 ? 4 : 2;          // what 227 KB hold of 512 threads' packets
    static constexpr int PACKETS = (RES ? 2 : 1) * 2 * Group8<T>::N;       // dy, residual; then 8 bytes of q and a scale for each group
    static constexpr size_t PER_THREAD = STAGES * (PACKETS * 16 + 2 * 8 + 2 * 4);
};
template <typename T, bool RES, bool AGAIN>
__global__ void __launch_bounds__(A8_LN_THREADS, 1)
a8_ln_bwd_kernel(const T* dy, const T* __restrict__ gamma, const T* __restrict__ beta, const float* __restrict__ var,
                 const int8_t* __restrict__ q, const float* __restrict__ scale, const T* residual, T* dx, T* __restrict__ y,
                 float* __restrict__ part, int64_t rows, int cols, int team) {
    using G = Group8<T>;
    using S = LnBwdSmem<T, RES>;
    extern __shared__ __align__(16) unsigned char ln_smem[];
    __shared__ float2 red[2][A8_LN_THREADS / 32];
    const int threads = blockDim.x;
    const int tid = threadIdx.x % team, group = threadIdx.x / team, groups = threads / team;
    const int c0 = tid * 8, c1 = (team + tid) * 8, blocks = (cols + A8_BLOCK - 1) / A8_BLOCK;
    const bool live0 = c0 < cols, live1 = c1 < cols;
    const float inv_n = 1.0f / (float)cols;
    float2* r0 = red[0] + group * (team >> 5);
    float2* r1 = red[1] + group * (team >> 5);
    uint4* const packets = reinterpret_cast<uint4*>(ln_smem) + threadIdx.x;                                                   // [stage][packet][thread]
    uint2* const bytes = reinterpret_cast<uint2*>(ln_smem + (size_t)threads * S::STAGES * S::PACKETS * 16) + threadIdx.x;       // [stage][group][thread]
    float* const scales = reinterpret_cast<float*>(ln_smem + (size_t)threads * S::STAGES * (S::PACKETS * 16 + 16)) + threadIdx.x;
    float2 dg[8], db[8], ga[8];
#pragma unroll
    for (int e = 0; e < 8; e++) dg[e] = db[e] = ga[e] = both(0.0f);
    if (live0) G::load(gamma + c0, ga);
    if (live1) G::load(gamma + c1, ga + 4);
    for (int i = 0; i < S::STAGES * S::PACKETS; i++)          // columns beyond the last stay zero
        if (!((i / G::N) & 1 ? live1 : live0)) packets[i * threads] = make_uint4(0, 0, 0, 0);
    for (int i = 0; i < S::STAGES * 2; i++) {
        if (i & 1 ? live1 : live0) continue;
        bytes[i * threads] = make_uint2(0, 0);
        scales[i * threads] = 0.0f;
    }
    pdl_wait();

    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + group;
    auto fetch = [&](int64_t r, int stage) {
        if (r < rows) {
            const int64_t at = r * cols;
            uint4* slot = packets + stage * S::PACKETS * threads;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int c = k ? c1 : c0;
                if (!(k ? live1 : live0)) continue;
                G::fetch(slot + k * G::N * threads, threads, dy + at + c);
                if (RES) G::fetch(slot + (2 + k) * G::N * threads, threads, residual + at + c);
                copy_async<8>(bytes + (stage * 2 + k) * threads, q + at + c);
                copy_async<4>(scales + (stage * 2 + k) * threads, scale + r * blocks + (c >> 7));
            }
        }
        copy_commit();
    };
    for (int i = 0; i < S::STAGES - 1; i++) fetch(row + i * step, i);
    float n_var = row < rows ? var[row] : 1.0f;
    for (int stage = 0, turn = 0; row < rows; row += step, turn ^= 1, stage = stage + 1 == S::STAGES ? 0 : stage + 1) {
        copy_wait<S::STAGES - 2>();
        fetch(row + (S::STAGES - 1) * step, stage == 0 ? S::STAGES - 1 : stage - 1);
        const float rstd = rsqrtf(n_var);
        if (row + step < rows) n_var = var[row + step];
        const uint4* slot = packets + stage * S::PACKETS * threads;
        const uint2 w0 = bytes[stage * 2 * threads], w1 = bytes[(stage * 2 + 1) * threads];
        const float s0 = scales[stage * 2 * threads], s1 = scales[(stage * 2 + 1) * threads];
        float2 a = both(0.0f), b = both(0.0f), g[8], xh[8];
        G::read(slot, threads, g);
        G::read(slot + G::N * threads, threads, g + 4);
        a8_unpack8(w0, s0, xh);
        a8_unpack8(w1, s1, xh + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            dg[e] = __ffma2_rn(g[e], xh[e], dg[e]);
            db[e] = __fadd2_rn(db[e], g[e]);
            g[e] = __fmul2_rn(g[e], ga[e]);
            a = __fadd2_rn(a, g[e]);
            b = __ffma2_rn(g[e], xh[e], b);
        }
        const float2 m = team_sum2(a.x + a.y, b.x + b.y, turn ? r1 : r0, group + 1, team);
        const float2 mg = both(-rstd * m.x * inv_n), mgx = both(-rstd * m.y * inv_n);
        const int64_t at = row * cols;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int c = k ? c1 : c0;
            if (!(k ? live1 : live0)) continue;
            float2 o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = __ffma2_rn(xh[4 * k + e], mgx, __ffma2_rn(g[4 * k + e], both(rstd), mg));
            if (RES) {
                float2 r[4];
                G::read(slot + (2 + k) * G::N * threads, threads, r);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = __fadd2_rn(o[e], r[e]);
            }
            G::write(dx + at + c, o);
            if (AGAIN) {
                float2 be[4];
                G::load(beta + c, be);                     // the same for every row: in the first-level cache
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = __ffma2_rn(xh[4 * k + e], ga[4 * k + e], be[e]);
                G::write(y + at + c, o);
            }
        }
    }
    copy_wait<0>();
    float* const fold = reinterpret_cast<float*>(ln_smem);          // [teams - 1][2][8 pairs][member]: the slots are done with
    if (groups > 1) {
        __syncthreads();
        float2* const mine = reinterpret_cast<float2*>(fold) + tid;
        if (group > 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                mine[((group - 1) * 16 + e) * team] = dg[e];
                mine[((group - 1) * 16 + 8 + e) * team] = db[e];
            }
        }
        __syncthreads();
        if (group == 0) {
            for (int k = 0; k < groups - 1; k++) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    dg[e] = __fadd2_rn(dg[e], mine[(k * 16 + e) * team]);
                    db[e] = __fadd2_rn(db[e], mine[(k * 16 + 8 + e) * team]);
                }
            }
        }
    }
    if (group == 0) {
        float* const p = part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int c = k ? c1 : c0;
            if (!(k ? live1 : live0)) continue;
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                *reinterpret_cast<float4*>(p + c + 2 * e) = make_float4(dg[4 * k + e].x, dg[4 * k + e].y, dg[4 * k + e + 1].x, dg[4 * k + e + 1].y);
                *reinterpret_cast<float4*>(p + cols + c + 2 * e) = make_float4(db[4 * k + e].x, db[4 * k + e].y, db[4 * k + e + 1].x, db[4 * k + e + 1].y);
            }
        }
    }
    pdl_launch_dependents();
}

// any column count and alignment: a CTA walks rows one at a time, scalar accesses, column sums in its row of `part`
template <typename T>
__global__ void __launch_bounds__(A8_THREADS)
a8_ln_bwd_generic_kernel(const T* dy, const T* gamma, const T* beta, const float* var, const int8_t* q, const float* scale, const T* residual,
                         T* dx, T* y, float* part, int64_t rows, int cols) {
    __shared__ float red[64];
    const int blocks = (cols + A8_BLOCK - 1) / A8_BLOCK;
    float* p = part + (int64_t)blockIdx.x * 2 * cols;
    for (int i = threadIdx.x; i < 2 * cols; i += A8_THREADS) p[i] = 0.0f;
    __syncthreads();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t at = row * cols;
        float a = 0.0f, b = 0.0f;
        for (int i = threadIdx.x; i < cols; i += A8_THREADS) {
            const float xh = (float)q[at + i] * scale[row * blocks + i / A8_BLOCK], d = to_f32(dy[at + i]), g = d * to_f32(gamma[i]);
            a += g;
            b = fmaf(g, xh, b);
            p[i] = fmaf(d, xh, p[i]);              // column i of this CTA's sums belongs to this thread in every row
            p[cols + i] += d;
        }
        block_sum2(a, b, red);
        const float mg = a / (float)cols, mgx = b / (float)cols, rstd = rsqrtf(var[row]);
        for (int i = threadIdx.x; i < cols; i += A8_THREADS) {
            const float xh = (float)q[at + i] * scale[row * blocks + i / A8_BLOCK], w = to_f32(gamma[i]);
            float o = rstd * (to_f32(dy[at + i]) * w - mg - xh * mgx);
            if (residual) o += to_f32(residual[at + i]);
            dx[at + i] = from_f32<T>(o);
            if (y) y[at + i] = from_f32<T>(fmaf(xh, w, to_f32(beta[i])));
        }
    }
}

// out[j] (+)= sum of part[k][j] in a fixed order: 32 columns per CTA, 8 warps take every 8th partial row each
template <typename T>
__global__ void __launch_bounds__(256)
a8_ln_reduce_kernel(const float* part, T* dgamma, T* dbeta, int parts, int cols, int accumulate) {
    __shared__ float s[8][33];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + lane;
    float a = 0.0f;
    if (j < 2 * (int64_t)cols) {
#pragma unroll 8
        for (int k = warp; k < parts; k += 8) a += part[(int64_t)k * 2 * cols + j];
    }
    s[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && j < 2 * (int64_t)cols) {
        for (int k = 1; k < 8; k++) a += s[k][lane];
        T* o = j < cols ? dgamma + j : dbeta + (j - cols);
        *o = from_f32<T>(accumulate ? to_f32(*o) + a : a);
    }
}

// threads that own a row of `cols` columns in the backward, 16 each
static int a8_team(int64_t cols) { return (int)((cols + 511) / 512) * 32; }

// more than the 48 KB of dynamic shared memory that need no leave
static cudaError_t a8_allow_smem(const void* kernel, size_t bytes) {
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

constexpr int A8_MAX_PARTS = 256;             // partial rows of the LayerNorm backward: one per CTA

template <typename T>
static int a8_ln_fwd(const void* x, const void* gamma, const void* beta, void* y, int8_t* q, float* scale, float* var, int64_t rows, int64_t cols,
                     float eps, cudaStream_t st) {
    if (cols % 16 == 0 && cols <= A8_LN_MAX_COLS && aligned16(x) && aligned16(gamma) && aligned16(beta) && aligned16(y) && aligned16(q)) {
        const int team = (int)((cols + 1023) / 1024) * 32, groups = LnFwd<T>::THREADS / team;       // 32 columns a thread
        const int64_t want = (rows + groups - 1) / groups, cap = (int64_t)sm_count() * LnFwd<T>::CTAS;
        const int grid = (int)(want < cap ? want : cap);
        const size_t smem = (size_t)team * groups * LnFwd<T>::PER_THREAD + (size_t)team * LnFwd<T>::PER_MEMBER;
        cudaError_t e = a8_allow_smem((const void*)a8_ln_fwd_kernel<T>, smem);
        if (e != cudaSuccess) {
            set_cuda_error(e, "a8_ln_fwd smem attribute");
            return BRK_CUDA_ERROR;
        }
        e = launch_pdl(a8_ln_fwd_kernel<T>, grid, team * groups, smem, st, (const T*)x, (const T*)gamma, (const T*)beta, (T*)y, q, scale, var, rows, (int)cols, eps, team);
        if (e != cudaSuccess) {
            set_cuda_error(e, "a8_ln_fwd_kernel");
            return BRK_CUDA_ERROR;
        }
        return launch_status("a8_ln_fwd_kernel");
    }
    a8_ln_fwd_generic_kernel<T><<<(unsigned)rows, A8_THREADS, 0, st>>>((const T*)x, (const T*)gamma, (const T*)beta, (T*)y, q, scale, var, (int)cols, eps);
    return launch_status("a8_ln_fwd_generic_kernel");
}

template <typename T, bool RES, bool AGAIN>
static cudaError_t a8_launch_ln_bwd(int grid, int block, cudaStream_t st, const T* dy, const T* gamma, const T* beta, const float* var,
                                    const int8_t* q, const float* scale, const T* residual, T* dx, T* y, float* part, int64_t rows, int cols, int team) {
    const size_t smem = (size_t)block * LnBwdSmem<T, RES>::PER_THREAD;
    static_assert(A8_LN_THREADS * LnBwdSmem<T, RES>::PER_THREAD <= 230000, "the slots must fit the 227 KB a CTA can have");
    static_assert(LnBwdSmem<T, RES>::PER_THREAD >= 128, "a team's column sums are folded in its slots");
    const cudaError_t e = a8_allow_smem((const void*)a8_ln_bwd_kernel<T, RES, AGAIN>, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(a8_ln_bwd_kernel<T, RES, AGAIN>, grid, block, smem, st, dy, gamma, beta, var, q, scale, residual, dx, y, part, rows, cols, team);
}

template <typename T>
static int a8_ln_bwd(const void* dy_, const void* gamma_, const void* beta_, const float* var, const int8_t* q, const float* scale, const void* residual_,
                     void* dgamma, void* dbeta, void* dx_, void* y_, int64_t rows, int64_t cols, float* part, int accumulate, cudaStream_t st) {
    const T *dy = (const T*)dy_, *gamma = (const T*)gamma_, *beta = (const T*)beta_, *residual = (const T*)residual_;
    T *dx = (T*)dx_, *y = (T*)y_;
    int parts;
    if (cols % 16 == 0 && cols <= A8_LN_MAX_COLS && aligned16(dy) && aligned16(gamma) && aligned16(dx) && aligned16(part) && (!residual || aligned16(residual)) &&
        (!y || (aligned16(y) && aligned16(beta))) && aligned16(q)) {
        const int team = a8_team(cols);
        int groups = A8_LN_THREADS / team;
        if ((int64_t)groups * sm_count() > rows) groups = (int)((rows + sm_count() - 1) / sm_count());      // few rows: spread them over the SMs
        if (groups > 15) groups = 15;                                                                      // named barriers 1..15
        const int64_t want = (rows + groups - 1) / groups;
        int grid = sm_count() < A8_MAX_PARTS ? sm_count() : A8_MAX_PARTS;
        if (want < grid) grid = (int)want;
        cudaError_t e;
        if (residual)
            e = y ? a8_launch_ln_bwd<T, true, true>(grid, team * groups, st, dy, gamma, beta, var, q, scale, residual, dx, y, part, rows, (int)cols, team)
                  : a8_launch_ln_bwd<T, true, false>(grid, team * groups, st, dy, gamma, beta, var, q, scale, residual, dx, y, part, rows, (int)cols, team);
        else
            e = y ? a8_launch_ln_bwd<T, false, true>(grid, team * groups, st, dy, gamma, beta, var, q, scale, residual, dx, y, part, rows, (int)cols, team)
                  : a8_launch_ln_bwd<T, false, false>(grid, team * groups, st, dy, gamma, beta, var, q, scale, residual, dx, y, part, rows, (int)cols, team);
        if (e != cudaSuccess) {
            set_cuda_error(e, "a8_ln_bwd_kernel");
            return BRK_CUDA_ERROR;
        }
        const int rc = launch_status("a8_ln_bwd_kernel");
        if (rc) return rc;
        parts = grid;
    } else {
        parts = (int)(rows < A8_MAX_PARTS ? rows : A8_MAX_PARTS);
        a8_ln_bwd_generic_kernel<T><<<parts, A8_THREADS, 0, st>>>(dy, gamma, beta, var, q, scale, residual, dx, y, part, rows, (int)cols);
        const int rc = launch_status("a8_ln_bwd_generic_kernel");
        if (rc) return rc;
    }
    const cudaError_t e = launch_pdl(a8_ln_reduce_kernel<T>, (int)((2 * cols + 31) / 32), 256, 0, st, (const float*)part, (T*)dgamma, (T*)dbeta, parts, (int)cols, accumulate);
    if (e != cudaSuccess) {
        set_cuda_error(e, "a8_ln_reduce_kernel");
        return BRK_CUDA_ERROR;
    }
    return launch_status("a8_ln_reduce_kernel");
}

static bool a8_sizes_ok(int64_t rows, int64_t cols) { return rows >= 0 && cols > 0 && rows <= 0x7fffffff && cols <= (1 << 24); }

}  // namespace brk

using namespace brk;

extern "C" int brk_act8_pack(const void* x, int8_t* q, float* scale, int64_t rows, int64_t cols, int dtype, void* stream) {
    if (!a8_sizes_ok(rows, cols)) return BRK_ATTR_ERROR;
    if (dtype != BRK_F32 && dtype != BRK_F16) return BRK_ATTR_ERROR;
    if (rows == 0) return BRK_OK;
    if (!x) return BRK_INPUT_ERROR;
    if (!q || !scale) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == BRK_F32) return a8_pack<float, false>(x, nullptr, q, scale, rows, cols, st);
    return a8_pack<__half, false>(x, nullptr, q, scale, rows, cols, st);
}

extern "C" int brk_act8_unpack(const int8_t* q, const float* scale, void* out, int64_t rows, int64_t cols, int dtype, void* stream) {
    if (!a8_sizes_ok(rows, cols)) return BRK_ATTR_ERROR;
    if (dtype != BRK_F32 && dtype != BRK_F16) return BRK_ATTR_ERROR;
    if (rows == 0) return BRK_OK;
    if (!q || !scale) return BRK_INPUT_ERROR;
    if (!out) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == BRK_F32) return a8_unpack<float, false>(q, scale, nullptr, out, nullptr, rows, cols, st);
    return a8_unpack<__half, false>(q, scale, nullptr, out, nullptr, rows, cols, st);
}

extern "C" int brk_gelu_fwd_act8(const void* x, void* y, int8_t* q, float* scale, int64_t rows, int64_t cols, int dtype, void* stream) {
    if (!a8_sizes_ok(rows, cols)) return BRK_ATTR_ERROR;
    if (dtype != BRK_F32 && dtype != BRK_F16) return BRK_ATTR_ERROR;
    if (rows == 0) return BRK_OK;
    if (!x) return BRK_INPUT_ERROR;
    if (!y || !q || !scale) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == BRK_F32) return a8_pack<float, true>(x, y, q, scale, rows, cols, st);
    return a8_pack<__half, true>(x, y, q, scale, rows, cols, st);
}

extern "C" int brk_gelu_bwd_act8(const void* dy, const int8_t* q, const float* scale, void* dx, void* y, int64_t rows, int64_t cols, int dtype, void* stream) {
    if (!a8_sizes_ok(rows, cols)) return BRK_ATTR_ERROR;
    if (dtype != BRK_F32 && dtype != BRK_F16) return BRK_ATTR_ERROR;
    if (rows == 0) return BRK_OK;
    if (!dy || !q || !scale) return BRK_INPUT_ERROR;
    if (!dx) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == BRK_F32) return a8_unpack<float, true>(q, scale, dy, dx, y, rows, cols, st);
    return a8_unpack<__half, true>(q, scale, dy, dx, y, rows, cols, st);
}

extern "C" int brk_layernorm_fwd_act8(const void* x, const void* gamma, const void* beta, void* y, int8_t* q, float* scale, float* var, int64_t rows,
                                      int64_t hidden, float eps, int dtype, void* stream) {
    if (!a8_sizes_ok(rows, hidden) || !(eps >= 0.0f)) return BRK_ATTR_ERROR;
    if (dtype != BRK_F32 && dtype != BRK_F16) return BRK_ATTR_ERROR;
    if (rows == 0) return BRK_OK;
    if (!x || !gamma || !beta) return BRK_INPUT_ERROR;
    if (!y || !q || !scale || !var) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == BRK_F32) return a8_ln_fwd<float>(x, gamma, beta, y, q, scale, var, rows, hidden, eps, st);
    return a8_ln_fwd<__half>(x, gamma, beta, y, q, scale, var, rows, hidden, eps, st);
}

extern "C" size_t brk_layernorm_bwd_act8_workspace_bytes(int64_t rows, int64_t hidden) {
    if (rows <= 0 || hidden <= 0) return 0;
    return (size_t)(rows < A8_MAX_PARTS ? rows : A8_MAX_PARTS) * 2 * (size_t)hidden * sizeof(float);
}

extern "C" int brk_layernorm_bwd_act8(const void* dy, const void* gamma, const void* beta, const float* var, const int8_t* q, const float* scale,
                                      const void* residual, void* dgamma, void* dbeta, void* dx, void* y, int64_t rows, int64_t hidden, void* workspace,
                                      size_t workspace_bytes, int accumulate, int dtype, void* stream) {
    if (!a8_sizes_ok(rows, hidden)) return BRK_ATTR_ERROR;
    if (dtype != BRK_F32 && dtype != BRK_F16) return BRK_ATTR_ERROR;
    if (!gamma || (y && !beta)) return BRK_INPUT_ERROR;
    if (!dgamma || !dbeta) return BRK_OUTPUT_ERROR;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {                          // no rows: the sums are zero
        if (accumulate) return BRK_OK;
        const size_t bytes = (size_t)hidden * (dtype == BRK_F32 ? 4 : 2);
        cudaError_t e = cudaMemsetAsync(dgamma, 0, bytes, st);
        if (e == cudaSuccess) e = cudaMemsetAsync(dbeta, 0, bytes, st);
        if (e != cudaSuccess) {
            set_cuda_error(e, "layernorm_bwd_act8 clear");
            return BRK_CUDA_ERROR;
        }
        return BRK_OK;
    }
    if (!dy || !var || !q || !scale) return BRK_INPUT_ERROR;
    if (!dx) return BRK_OUTPUT_ERROR;
    if (!workspace || workspace_bytes < brk_layernorm_bwd_act8_workspace_bytes(rows, hidden) || (reinterpret_cast<uintptr_t>(workspace) & 3)) return BRK_ATTR_ERROR;
    if (dtype == BRK_F32) return a8_ln_bwd<float>(dy, gamma, beta, var, q, scale, residual, dgamma, dbeta, dx, y, rows, hidden, (float*)workspace, accumulate, st);
    return a8_ln_bwd<__half>(dy, gamma, beta, var, q, scale, residual, dgamma, dbeta, dx, y, rows, hidden, (float*)workspace, accumulate, st);
}
