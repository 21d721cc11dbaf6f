// Dropout whose mask is a function of (seed, step, element index) and is never stored:
//     out_i = [residual_i +] (keep_i ? x_i / (1 - p) : 0),     keep_i = word_i >= round(p 2^32)
// word_i is word (i mod 4) of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel Random Numbers: As Easy as 1, 2, 3",
// SC'11) with the counter (i div 4, step) and the key seed, and i the element's row-major index, so the mask depends
// neither on the strides nor on the launch.  The backward pass is the same call on the gradient.
//
// Not part of the reference.  In a training step it drops whole splats: their opacities go through it, which is how
// ViewRenderer.render_views applies it.
//
// A dropped element is selected away, not multiplied by zero, so an infinity or NaN in it leaves no trace.  The product
// and the residual's addition are one fused multiply-add in 32 bits, rounded once to the storage type.
#include <cmath>

#include "vector_io.cuh"

namespace dsb {

namespace {

constexpr int kThreads = 256;

struct DropoutArgs {
    long long count, cols, x_stride, residual_stride, out_stride;
    u32 threshold;
    int drop_all;              // p = 1: the threshold 2^32 does not fit a word
    float scale;
    u32 seed_lo, seed_hi, step_lo, step_hi;
    const long long* rng;      // (seed, step) on the device, or null
    long long* rng_used;       // where the pair that was used is written down, or null
};

__device__ __forceinline__ uint4 philox4x32_10(u32 c0, u32 c1, u32 c2, u32 c3, u32 k0, u32 k1) {
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const u64 p0 = (u64)0xD2511F53u * c0, p1 = (u64)0xCD9E8D57u * c2;
        c0 = (u32)(p1 >> 32) ^ c1 ^ k0;
        c1 = (u32)p1;
        c2 = (u32)(p0 >> 32) ^ c3 ^ k1;
        c3 = (u32)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

template <int V>
__device__ __forceinline__ void philox_words_at(u64 first_block, u32 step_lo, u32 step_hi, u32 seed_lo, u32 seed_hi, u32 (&word)[V]) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        const u64 block = first_block + q;
        const uint4 w = philox4x32_10((u32)block, (u32)(block >> 32), step_lo, step_hi, seed_lo, seed_hi);
        word[4 * q] = w.x; word[4 * q + 1] = w.y; word[4 * q + 2] = w.z; word[4 * q + 3] = w.w;
    }
}

// Each thread takes V consecutive elements a trip (V a multiple of 4: whole counter blocks).  VEC: they lie in one row, at
// addresses that allow one transaction; else every element finds its own row.  The loads of a trip are issued before its
// random words are worked out.  What bounds it, on tensors of 168 MB: with 32-bit ones memory (77 us with a residual, 59 without,
// 1.0 and 0.87 of the copy rate).  With 16-bit ones, twice the elements, 85 us with and without: the generator, in 22 instructions an
// element, but no unit of the GPU is full.  Issue slots are busy for 64% of the time; the five 32 x 32 -> 64 bit products an
// element, at four cycles each, keep the multiplier busy for half of it (45 us); DRAM 33% (58% with a residual).  Six blocks an SM
// (40 registers) were the fastest of 4, 6 and 8; one trip per thread instead of a few loses a fifth.
template <typename T, int V, bool VEC, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads, 6)
dropout_kernel(const T* x, const T* residual, T* out, const DropoutArgs a) {
    u32 seed_lo = a.seed_lo, seed_hi = a.seed_hi, step_lo = a.step_lo, step_hi = a.step_hi;
    if (a.rng) {
        const u64 seed = (u64)a.rng[0], step = (u64)a.rng[1];
        seed_lo = (u32)seed; seed_hi = (u32)(seed >> 32); step_lo = (u32)step; step_hi = (u32)(step >> 32);
        if (a.rng_used && blockIdx.x == 0 && threadIdx.x == 0) { a.rng_used[0] = (long long)seed; a.rng_used[1] = (long long)step; }
    }
    const u32 threshold = a.threshold;
    const float scale = a.scale;
    const long long stride = (long long)gridDim.x * kThreads * V;
    const bool flat = a.x_stride == a.cols && a.residual_stride == a.cols && a.out_stride == a.cols;
    long long i = ((long long)blockIdx.x * kThreads + threadIdx.x) * V;
    if (VEC) {
        for (; i + V <= a.count; i += stride) {
            long long row = 0, col = i;
            if (!flat) { row = i / a.cols; col = i - row * a.cols; }
            const Pack<T, V> xv = load_pack<T, V>(x + row * a.x_stride + col);
            Pack<T, V> rv;
            if (RESIDUAL) rv = load_pack<T, V>(residual + row * a.residual_stride + col);
            u32 word[V];
            philox_words_at<V>((u64)(i >> 2), step_lo, step_hi, seed_lo, seed_hi, word);
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float v = to_float(xv.e[e]), r = RESIDUAL ? to_float(rv.e[e]) : 0.f;
                o[e] = word[e] >= threshold && !a.drop_all ? (RESIDUAL ? fmaf(v, scale, r) : v * scale) : r;
            }
            store_floats<T, V>(out + row * a.out_stride + col, o);
        }
    }
    for (; i < a.count; i += stride) {
        u32 word[V];
        philox_words_at<V>((u64)(i >> 2), step_lo, step_hi, seed_lo, seed_hi, word);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const long long at = i + e;
            if (at >= a.count) break;
            const long long row = flat ? 0 : at / a.cols, col = at - row * a.cols;
            const float v = to_float(x[row * a.x_stride + col]), r = RESIDUAL ? to_float(residual[row * a.residual_stride + col]) : 0.f;
            const float o = word[e] >= threshold && !a.drop_all ? (RESIDUAL ? fmaf(v, scale, r) : v * scale) : r;
            from_float(o, out[row * a.out_stride + col]);
        }
    }
}

}  // namespace

int launch_dropout(const void* x, const void* residual, void* out, int64_t rows, int64_t cols, int64_t x_stride,
                   int64_t residual_stride, int64_t out_stride, int dtype, double p, uint64_t seed, uint64_t step,
                   const int64_t* rng, int64_t* rng_used, cudaStream_t s) {
    DSB_REQUIRE(rows >= 0 && cols >= 0 && (cols == 0 || rows <= ((int64_t)1 << 60) / cols), "dropout: bad size");
    DSB_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: p must lie in [0, 1]");
    DSB_REQUIRE(dtype == DSB_DTYPE_F32 || dtype == DSB_DTYPE_F16 || dtype == DSB_DTYPE_BF16, "dropout: unknown dtype %d", dtype);
    if (rows == 0 || cols == 0) return DSB_OK;
    DSB_REQUIRE(x && out, "dropout: null pointer");
    const double edge = std::nearbyint(p * 4294967296.0);   // the product is exact; ties to even
    DropoutArgs a;
    a.drop_all = edge >= 4294967296.0;
    a.threshold = a.drop_all ? 0xffffffffu : (u32)edge;
    a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
    a.count = rows * cols; a.cols = cols;
    if (rows == 1) x_stride = residual_stride = out_stride = cols;   // a row's stride says nothing then
    if (!residual) residual_stride = cols;
    a.x_stride = x_stride; a.residual_stride = residual_stride; a.out_stride = out_stride;
    a.seed_lo = (u32)seed; a.seed_hi = (u32)(seed >> 32); a.step_lo = (u32)step; a.step_hi = (u32)(step >> 32);
    a.rng = reinterpret_cast<const long long*>(rng); a.rng_used = reinterpret_cast<long long*>(rng_used);
    with_dtype(dtype, [&](auto tag) {
        typedef decltype(tag) T;
        constexpr int V = 16 / sizeof(T);
        const bool flat = x_stride == cols && residual_stride == cols && out_stride == cols;
        bool vec = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)out) & 15) == 0;
        if (!flat) vec = vec && ((cols | x_stride | residual_stride | out_stride) % V) == 0;
        long long blocks = ((a.count + V - 1) / V + kThreads - 1) / kThreads;
        if (blocks > 148 * 16) blocks = 148 * 16;   // grid-stride loop beyond sixteen blocks per SM
        const T* tx = static_cast<const T*>(x);
        const T* tr = static_cast<const T*>(residual);
        T* to = static_cast<T*>(out);
        auto launch = [&](auto kernel) { kernel<<<(unsigned)blocks, kThreads, 0, s>>>(tx, tr, to, a); };
        if (vec && tr) launch(dropout_kernel<T, V, true, true>);
        else if (vec) launch(dropout_kernel<T, V, true, false>);
        else if (tr) launch(dropout_kernel<T, V, false, true>);
        else launch(dropout_kernel<T, V, false, false>);
    });
    DSB_LAUNCH_CHECK();
    return DSB_OK;
}

}  // namespace dsb
