// Gated linear recurrence over sequences, forward and backward, and its single-row form:
//     f_t = gate_t or 1 / (1 + exp(-gate_t)),   h_t = f_t h_{t-1} + i_t,   i_t = x_t or, coupled, (1 - f_t) x_t
//     g_t = v_h_t + q_{t+1},   q_t = f_t g_t,   v_x_t = g_t or (1 - f_t) g_t
//     v_f_t = sum over the channels that share the gate of g_t (h_{t-1}, coupled: h_{t-1} - x_t),   v_state_in = q_0
// Not part of the reference as an operator of its own; its blend (cpp/rasterizer_kernels.cu:341-431) is the coupled form
// over a tile's list, back to front, with f = 1 - alpha.
//
// A stretch of rows maps the state before it to the state after it as h -> a h + b, and two stretches compose as
// (a2 a1, a2 b1 + b2); a stretch in which a sequence begins maps every h to b ("closed": its a is never looked at, so
// that an infinity of the sequence before cannot meet a zero).  Rows are cut into chunks of a tile's rows, channels into
// blocks; a tile's thread runs L consecutive rows of V channels, the warp composes its threads' maps, the block its warps'.
//   1. aggregate: every tile's map
//   2. carry:     one thread per sequence chain and channel walks the chunks' maps and leaves the state before each chunk
//   3. apply:     every tile again, now with the state it starts from
// The backward runs the same three steps from the last row to the first on q, and recomputes h inside a tile from the
// state its chunk starts with (a checkpoint of the forward), in 32 bits: the h that was written out is rounded to the
// storage type and need not be kept.
#include <type_traits>

#include "vector_io.cuh"

namespace dsb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr long long kMaxRows = (1ll << 31) - 1;

struct Layout {            // how a call is cut; the same for the forward and the backward of one shape
    int vec;               // channels per thread: 4 or 1
    int lg_tx;             // log2 of the threads side by side on one row
    int per_head;          // channels that share a gate; all of them when every channel has its own
    int heads;             // 1 when every channel has its own gate
    int parts;             // channel blocks per head
    bool table;            // chunks may hold sequence borders: one chain over all rows; else one chain per sequence
    long long chains, chain_rows;
};

struct Args {
    const void *x, *gate, *v_h;
    void *h, *v_x, *v_gate;
    const float *state_in, *v_state_out;
    float *state_out, *v_state_in;
    float* checkpoints;
    float *map_a, *map_b;  // [chains][chunks][channels]; map_a becomes the state before each chunk
    int* map_closed;       // [chains][chunks]
    float* gate_parts;     // [parts][rows][heads], when a head spans several channel blocks
    const int *offsets, *lengths;
    int* device_status;
    long long rows, chain_rows, chains;
    long long x_stride, gate_stride, v_h_stride;   // negative when the scan runs from the last row to the first
    long long h_stride, gate_out_stride;           // channels / heads of contiguous results, with the same sign
    long long chunks, checkpoint_chunks;
    int checkpoint_rows;
    int sequences, sequence_rows, channels, gate_heads, heads, per_head, parts, lg_tx;
    int logit, coupled, reverse, shared;
};

// ---- gates ---------------------------------------------------------------------------------------------------------
// One register holds both f and 1 - f to full relative precision where they are small: for a logit the smaller of the two,
// m = exp(-|g|) / (1 + exp(-|g|)) <= 1/2, with the sign saying which one it is.
__device__ __forceinline__ float encode_gate(float g, int logit) {
    if (!logit) return g;
    const float y = -fabsf(g);
    // exp(y) = 2^(y log2 e): the product's rounding error and the constant's own are added back to first order
    const float hi = y * 1.44269502f;
    const float lo = fmaf(y, 1.92596303e-8f, fmaf(y, 1.44269502f, -hi));
    float t = exp2f(hi);
    t = y < -80.f ? t : fmaf(t, lo * 0.693147181f, t);   // beyond, t is 0 beside 1 (and lo is NaN at infinity)
    const float d = 1.f + t;
    float r = __fdividef(1.f, d);
    r = fmaf(r, fmaf(-d, r, 1.f), r);                     // one Newton step: 1 / d to rounding
    return copysignf(t * r, g);
}
__device__ __forceinline__ float gate_f(float m, int logit) {
    return logit ? (signbit(m) ? -m : 1.f - m) : m;
}
__device__ __forceinline__ float gate_k(float m, int logit) {   // 1 - f
    return logit ? (signbit(m) ? 1.f + m : m) : 1.f - m;
}

// ---- which rows begin and end sequences ------------------------------------------------------------------------------
constexpr int kNone = -1, kOutside = -2;

struct ChainRows {         // without a table: the chain is one sequence
    int sequence;
    long long lo, hi;      // the positions that belong to it
};
__device__ __forceinline__ ChainRows chain_rows_of(const Args& a, int chain) {
    ChainRows c;
    c.sequence = a.reverse ? a.sequences - 1 - chain : chain;
    long long len = a.sequence_rows;
    if (a.lengths) len = min(max(a.lengths[c.sequence], 0), a.sequence_rows);
    c.lo = a.reverse ? a.sequence_rows - len : 0;
    c.hi = c.lo + len;
    return c;
}

// How many of offsets[0 .. n) are <= row; called by one whole warp.
__device__ __forceinline__ int count_not_above(const int* offsets, int n, long long row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;
    while (len > 0) {
        const int step = (len + 31) / 32;
        const long long at = (long long)lane * step;
        const bool below = at < len && offsets[lo + at] <= row;
        const int below_count = __popc(__ballot_sync(0xffffffffu, below));
        if (below_count == 0) break;
        const int skip = (below_count - 1) * step + 1;
        len = min(step - 1, len - skip);
        lo += skip;
    }
    return lo;
}

// first[r] / end[r]: the sequence that begins / ends at position p0 + r, kNone, or (first only) kOutside.
__device__ void fill_row_table(const Args& a, long long p0, int tile_rows, int* first, int* end, int* s_seq) {
    const int tid = threadIdx.x;
    if (a.sequence_rows > 0) {
        for (int r = tid; r < tile_rows; r += kThreads) {
            const long long p = p0 + r;
            int f = kOutside, e = kNone;
            if (p < a.rows) {
                const int turn = (int)(p / a.sequence_rows), t = (int)(p - (long long)turn * a.sequence_rows);
                const int seq = a.reverse ? a.sequences - 1 - turn : turn;
                const int len = a.lengths ? min(max(a.lengths[seq], 0), a.sequence_rows) : a.sequence_rows;
                const int lo = a.reverse ? a.sequence_rows - len : 0;
                if (t >= lo && t < lo + len) {
                    f = t == lo ? seq : kNone;
                    e = t == lo + len - 1 ? seq : kNone;
                }
            }
            first[r] = f;
            end[r] = e;
        }
    } else {
        const long long p1 = min(p0 + tile_rows, a.rows);
        const long long row0 = a.reverse ? a.rows - p1 : p0, row1 = a.reverse ? a.rows - p0 : p1;
        const long long all0 = a.offsets[0], all1 = a.offsets[a.sequences];
        for (int r = tid; r < tile_rows; r += kThreads) {
            const long long p = p0 + r, row = a.reverse ? a.rows - 1 - p : p;
            first[r] = p < p1 && row >= all0 && row < all1 ? kNone : kOutside;
            end[r] = kNone;
        }
        if (tid < 32) {
            const int n = count_not_above(a.offsets, a.sequences, row0);
            if (tid == 0) *s_seq = max(n - 1, 0);
        }
        __syncthreads();
        for (int s = *s_seq + tid; s < a.sequences; s += kThreads) {
            const long long o0 = a.offsets[s], o1 = a.offsets[s + 1];
            if (o0 >= row1) break;
            if (o0 >= o1) continue;
            const long long front = a.reverse ? o1 - 1 : o0, back = a.reverse ? o0 : o1 - 1;
            if (front >= row0 && front < row1) {
                const int r = (int)(a.reverse ? row1 - 1 - front : front - row0);
                first[r] = s;
            }
            if (back >= row0 && back < row1) {
                const int r = (int)(a.reverse ? row1 - 1 - back : back - row0);
                end[r] = s;
            }
        }
    }
    __syncthreads();
}

// Sequences without rows hand their state on; offsets and lengths out of order or range are reported.
__device__ void pass_empty_sequences(const Args& a, const float* in, float* out) {
    if (!a.offsets && !a.lengths) return;
    const long long step = (long long)gridDim.x * kThreads;
    for (long long s = (long long)blockIdx.x * kThreads + threadIdx.x; s < a.sequences; s += step) {
        bool empty, bad;
        if (a.offsets) {
            const long long o0 = a.offsets[s], o1 = a.offsets[s + 1];
            empty = o1 <= o0;
            bad = o1 < o0 || o0 < 0 || o1 > a.rows;
        } else {
            const int len = a.lengths[s];
            empty = len <= 0;
            bad = len < 0 || len > a.sequence_rows;
        }
        if (bad) atomicMin(a.device_status, DSB_ERR_INVALID_ARGUMENT);
        if ((empty || bad) && out)
            for (int c = 0; c < a.channels; ++c) out[s * a.channels + c] = in ? in[s * a.channels + c] : 0.f;
    }
}

// ---- maps and their composition ----------------------------------------------------------------------------------------
template <int V>
struct Map {
    float a[V], b[V];
    int closed;
};
template <int V>
__device__ __forceinline__ void identity(Map<V>& m) {
#pragma unroll
    for (int v = 0; v < V; ++v) { m.a[v] = 1.f; m.b[v] = 0.f; }
    m.closed = 0;
}
// m <- m after e (e comes first along the scan)
template <int V>
__device__ __forceinline__ void compose_after(Map<V>& m, const Map<V>& e) {
    if (m.closed) return;
#pragma unroll
    for (int v = 0; v < V; ++v) { m.b[v] = fmaf(m.a[v], e.b[v], m.b[v]); m.a[v] *= e.a[v]; }
    m.closed = e.closed;
}
template <int V>
__device__ __forceinline__ void apply_map(float (&h)[V], const Map<V>& m) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = m.closed ? m.b[v] : fmaf(m.a[v], h[v], m.b[v]);
}

template <int V>
struct Shared {
    float a[kWarps][32 * V], b[kWarps][32 * V];
    int closed[kWarps];
    int seq;
};

// Lanes that hold the same channels on consecutive row groups are tx apart.  From every thread's own map `m`:
// the warp's running composition, its total in shared memory, and the map of the warp's rows before this thread's.
// FORWARD: rows run with the lane; else against it.
template <int V, bool FORWARD>
__device__ __forceinline__ Map<V> compose_warp(const Map<V>& own, int lg_tx, Shared<V>& sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tx = 1 << lg_tx;
    Map<V> run = own;
    for (int off = tx; off < 32; off <<= 1) {
        Map<V> e;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            e.a[v] = FORWARD ? __shfl_up_sync(0xffffffffu, run.a[v], off) : __shfl_down_sync(0xffffffffu, run.a[v], off);
            e.b[v] = FORWARD ? __shfl_up_sync(0xffffffffu, run.b[v], off) : __shfl_down_sync(0xffffffffu, run.b[v], off);
        }
        e.closed = FORWARD ? __shfl_up_sync(0xffffffffu, run.closed, off) : __shfl_down_sync(0xffffffffu, run.closed, off);
        if (FORWARD ? lane >= off : lane + off < 32) compose_after(run, e);
    }
    if (FORWARD ? lane >= 32 - tx : lane < tx) {
        const int at = (lane & (tx - 1)) * V;
#pragma unroll
        for (int v = 0; v < V; ++v) { sh.a[warp][at + v] = run.a[v]; sh.b[warp][at + v] = run.b[v]; }
        if ((lane & (tx - 1)) == 0) sh.closed[warp] = run.closed;
    }
    Map<V> before;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        before.a[v] = FORWARD ? __shfl_up_sync(0xffffffffu, run.a[v], tx) : __shfl_down_sync(0xffffffffu, run.a[v], tx);
        before.b[v] = FORWARD ? __shfl_up_sync(0xffffffffu, run.b[v], tx) : __shfl_down_sync(0xffffffffu, run.b[v], tx);
    }
    before.closed = FORWARD ? __shfl_up_sync(0xffffffffu, run.closed, tx) : __shfl_down_sync(0xffffffffu, run.closed, tx);
    if (FORWARD ? lane < tx : lane >= 32 - tx) identity(before);
    return before;
}
template <int V>
__device__ __forceinline__ Map<V> warp_total(const Shared<V>& sh, int warp, int tx) {
    Map<V> m;
#pragma unroll
    for (int v = 0; v < V; ++v) { m.a[v] = sh.a[warp][tx * V + v]; m.b[v] = sh.b[warp][tx * V + v]; }
    m.closed = sh.closed[warp];
    return m;
}

// ---- a tile's place ------------------------------------------------------------------------------------------------
struct Place {
    int chain, head, part, channel, tx;
    long long chunk, p0;
    int row0;              // this thread's first row inside the tile
    bool active;
    ChainRows rows;
};
template <int V, int L>
__device__ __forceinline__ Place place_of(const Args& a, long long tile, int tile_rows, bool table) {
    Place p;
    const int blocks = a.heads * a.parts;
    const int block = (int)(tile % blocks);
    const long long rest = tile / blocks;
    p.chain = (int)(rest % a.chains);
    p.chunk = rest / a.chains;
    p.p0 = p.chunk * tile_rows;
    p.head = block / a.parts;
    p.part = block - p.head * a.parts;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    p.tx = lane & ((1 << a.lg_tx) - 1);
    p.row0 = (warp * (32 >> a.lg_tx) + (lane >> a.lg_tx)) * L;
    const int c = (p.part << a.lg_tx) * V + p.tx * V;
    p.active = c < a.per_head;
    p.channel = p.head * a.per_head + c;
    if (!table) p.rows = chain_rows_of(a, p.chain);
    return p;
}
// The sequence that begins at the thread's row l (kNone, kOutside), and the one that ends there.
template <bool TABLE>
__device__ __forceinline__ int first_at(const Place& p, const int* table, int l) {
    if (TABLE) return table[p.row0 + l];
    const long long t = p.p0 + p.row0 + l;
    return t < p.rows.lo || t >= p.rows.hi ? kOutside : t == p.rows.lo ? p.rows.sequence : kNone;
}
template <bool TABLE>
__device__ __forceinline__ int end_at(const Place& p, const int* table, int l) {
    if (TABLE) return table[p.row0 + l];
    return p.p0 + p.row0 + l == p.rows.hi - 1 ? p.rows.sequence : kNone;
}

template <int V>
__device__ __forceinline__ void load_state(const float* states, long long index, int channels, int channel, float (&o)[V]) {
    if (!states) {
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = 0.f;
        return;
    }
    const Pack<float, V> q = load_pack<float, V>(states + index * channels + channel);
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = q.e[v];
}

// The thread's rows of x and the gate, all loads in flight together: x as floats, the gate encoded.  Rows that belong to no
// sequence: x = 0 and, whatever the form, a map that leaves the state as it is is the caller's business.
template <typename T, int V, int L, bool TABLE>
__device__ __forceinline__ void load_rows(const Args& a, const Place& p, const int* first, float (&x)[L][V], float (&m)[L][V]) {
    const T* px = static_cast<const T*>(a.x) + (p.chain * a.chain_rows + p.p0 + p.row0) * a.x_stride + p.channel;
    const T* pg = static_cast<const T*>(a.gate) + (p.chain * a.chain_rows + p.p0 + p.row0) * a.gate_stride +
                  (a.shared ? p.head : p.channel);
    Pack<T, V> rx[L], rg[L];
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const bool there = p.active && first_at<TABLE>(p, first, l) != kOutside;
        if (there) {
            rx[l] = load_pack<T, V>(px + l * a.x_stride);
            if (a.shared) rg[l].e[0] = pg[l * a.gate_stride];
            else rg[l] = load_pack<T, V>(pg + l * a.gate_stride);
        } else {
            memset(&rx[l], 0, sizeof(rx[l]));
            memset(&rg[l], 0, sizeof(rg[l]));
        }
    }
#pragma unroll
    for (int l = 0; l < L; ++l) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[l][v] = to_float(rx[l].e[v]);
            if (a.shared) m[l][v] = v == 0 ? encode_gate(to_float(rg[l].e[0]), a.logit) : m[l][0];
            else m[l][v] = encode_gate(to_float(rg[l].e[v]), a.logit);
        }
    }
}

template <typename T, int V, int L, bool TABLE, bool APPLY>
__global__ void __launch_bounds__(kThreads)
recurrence_forward_kernel(const Args a) {
    __shared__ Shared<V> sh;
    extern __shared__ int s_table[];
    const int tile_rows = kWarps * (32 >> a.lg_tx) * L;
    int* first = s_table;
    int* end = s_table + tile_rows;
    const Place p = place_of<V, L>(a, blockIdx.x, tile_rows, TABLE);
    if (TABLE) fill_row_table(a, p.p0, tile_rows, first, end, &sh.seq);
    float f[L][V], b[L][V];
    load_rows<T, V, L, TABLE>(a, p, first, b, f);

    Map<V> own;
    identity(own);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const int s = first_at<TABLE>(p, first, l);
        float st[V];
        if (s >= 0 && p.active) load_state<V>(a.state_in, s, a.channels, p.channel, st);
        if (s >= 0) own.closed = 1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float m = f[l][v];
            f[l][v] = s == kOutside ? 1.f : gate_f(m, a.logit);
            if (a.coupled) b[l][v] *= gate_k(m, a.logit);
            own.b[v] = fmaf(f[l][v], s >= 0 && p.active ? st[v] : own.b[v], b[l][v]);
            own.a[v] *= f[l][v];
        }
    }
    const Map<V> before = compose_warp<V, true>(own, a.lg_tx, sh);
    __syncthreads();
    const int warp = threadIdx.x >> 5;
    const long long at = (p.chain * a.chunks + p.chunk) * a.channels + p.channel;
    if (!APPLY) {
        if (warp == 0 && (threadIdx.x & 31) < (1 << a.lg_tx) && p.active) {
            Map<V> all = warp_total<V>(sh, kWarps - 1, p.tx);
            for (int w = kWarps - 2; w >= 0; --w) compose_after(all, warp_total<V>(sh, w, p.tx));
            store_floats<float, V>(a.map_a + at, all.a);
            store_floats<float, V>(a.map_b + at, all.b);
            if (p.tx == 0) a.map_closed[p.chain * a.chunks + p.chunk] = all.closed;
        }
        return;
    }
    float h[V];
    load_state<V>(p.active && a.chunks > 1 ? a.map_a : nullptr, p.chain * a.chunks + p.chunk, a.channels, p.channel, h);
    for (int w = 0; w < warp; ++w) apply_map(h, warp_total<V>(sh, w, p.tx));
    apply_map(h, before);
    const long long p_first = p.p0 + p.row0;
    if (a.checkpoints && p.active && p_first < a.chain_rows && p_first % a.checkpoint_rows == 0)
        store_floats<float, V>(a.checkpoints + (p.chain * a.checkpoint_chunks + p_first / a.checkpoint_rows) * a.channels + p.channel, h);
    T* ph = a.h ? static_cast<T*>(a.h) + (p.chain * a.chain_rows + p_first) * a.h_stride + p.channel : nullptr;
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const int s = first_at<TABLE>(p, first, l), e = end_at<TABLE>(p, end, l);
        if (s >= 0 && p.active) load_state<V>(a.state_in, s, a.channels, p.channel, h);
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = fmaf(f[l][v], h[v], b[l][v]);
            o[v] = s == kOutside ? 0.f : h[v];
        }
        if (ph && p.active && p_first + l < a.chain_rows) store_floats<T, V>(ph + l * a.h_stride, o);
        if (e >= 0 && p.active) store_floats<float, V>(a.state_out + (long long)e * a.channels + p.channel, h);
    }
    pass_empty_sequences(a, a.state_in, a.state_out);
}

// From the chunks' maps to the state before each chunk (after it, when the scan runs against the chunks).
template <bool FORWARD>
__global__ void __launch_bounds__(kThreads) recurrence_carry_kernel(const Args a) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= a.chains * a.channels) return;
    const long long chain = i / a.channels;
    const int c = (int)(i - chain * a.channels);
    float s = 0.f;
    for (long long j = 0; j < a.chunks; ++j) {
        const long long chunk = chain * a.chunks + (FORWARD ? j : a.chunks - 1 - j);
        const float ma = a.map_a[chunk * a.channels + c], mb = a.map_b[chunk * a.channels + c];
        a.map_a[chunk * a.channels + c] = s;
        s = a.map_closed[chunk] ? mb : fmaf(ma, s, mb);
    }
}

template <typename T, int V, int L, bool TABLE, bool APPLY>
__global__ void __launch_bounds__(kThreads)
recurrence_backward_kernel(const Args a) {
    __shared__ Shared<V> sh;
    extern __shared__ int s_table[];
    const int tile_rows = kWarps * (32 >> a.lg_tx) * L;
    int* first = s_table;
    int* end = s_table + tile_rows;
    const Place p = place_of<V, L>(a, blockIdx.x, tile_rows, TABLE);
    if (TABLE) fill_row_table(a, p.p0, tile_rows, first, end, &sh.seq);
    const int warp = threadIdx.x >> 5;
    const long long p_first = p.p0 + p.row0;
    float u[L][V], m[L][V], d[L][V];
    {
        const T* pd = static_cast<const T*>(a.v_h) + (p.chain * a.chain_rows + p_first) * a.v_h_stride + p.channel;
        Pack<T, V> rd[L];
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const bool there = a.v_h && p.active && first_at<TABLE>(p, first, l) != kOutside;
            if (there) rd[l] = load_pack<T, V>(pd + l * a.v_h_stride);
            else memset(&rd[l], 0, sizeof(rd[l]));
        }
        load_rows<T, V, L, TABLE>(a, p, first, u, m);
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
            for (int v = 0; v < V; ++v) d[l][v] = to_float(rd[l].e[v]);
    }
    if (APPLY) {   // u_t <- h_{t-1}, coupled: h_{t-1} - x_t
        Map<V> own;
        identity(own);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int s = first_at<TABLE>(p, first, l);
            float st[V];
            if (s >= 0 && p.active) load_state<V>(a.state_in, s, a.channels, p.channel, st);
            if (s >= 0) own.closed = 1;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float f = s == kOutside ? 1.f : gate_f(m[l][v], a.logit);
                const float b = a.coupled ? u[l][v] * gate_k(m[l][v], a.logit) : u[l][v];
                own.b[v] = fmaf(f, s >= 0 && p.active ? st[v] : own.b[v], b);
                own.a[v] *= f;
            }
        }
        const Map<V> before = compose_warp<V, true>(own, a.lg_tx, sh);
        __syncthreads();
        float h[V];
        load_state<V>(p.active && p.chunk > 0 ? a.checkpoints : nullptr, p.chain * a.checkpoint_chunks + p.chunk, a.channels,
                      p.channel, h);
        for (int w = 0; w < warp; ++w) apply_map(h, warp_total<V>(sh, w, p.tx));
        apply_map(h, before);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int s = first_at<TABLE>(p, first, l);
            if (s >= 0 && p.active) load_state<V>(a.state_in, s, a.channels, p.channel, h);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float f = s == kOutside ? 1.f : gate_f(m[l][v], a.logit);
                const float x = u[l][v];
                const float b = a.coupled ? x * gate_k(m[l][v], a.logit) : x;
                u[l][v] = a.coupled ? h[v] - x : h[v];
                h[v] = fmaf(f, h[v], b);
            }
        }
        __syncthreads();   // the warps' totals are about to be overwritten
    }
    Map<V> own;
    identity(own);
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
        const int s = first_at<TABLE>(p, first, l), e = end_at<TABLE>(p, end, l);
        float q[V];
        if (e >= 0 && p.active) load_state<V>(a.v_state_out, e, a.channels, p.channel, q);
        if (e >= 0) own.closed = 1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float f = s == kOutside ? 1.f : gate_f(m[l][v], a.logit);
            own.b[v] = f * (d[l][v] + (e >= 0 && p.active ? q[v] : own.b[v]));
            own.a[v] *= f;
        }
    }
    const Map<V> after = compose_warp<V, false>(own, a.lg_tx, sh);
    __syncthreads();
    const long long at = (p.chain * a.chunks + p.chunk) * a.channels + p.channel;
    if (!APPLY) {
        if (warp == 0 && (threadIdx.x & 31) < (1 << a.lg_tx) && p.active) {
            Map<V> all = warp_total<V>(sh, 0, p.tx);
            for (int w = 1; w < kWarps; ++w) compose_after(all, warp_total<V>(sh, w, p.tx));
            store_floats<float, V>(a.map_a + at, all.a);
            store_floats<float, V>(a.map_b + at, all.b);
            if (p.tx == 0) a.map_closed[p.chain * a.chunks + p.chunk] = all.closed;
        }
        return;
    }
    float q[V];
    load_state<V>(p.active && a.chunks > 1 ? a.map_a : nullptr, p.chain * a.chunks + p.chunk, a.channels, p.channel, q);
    for (int w = kWarps - 1; w > warp; --w) apply_map(q, warp_total<V>(sh, w, p.tx));
    apply_map(q, after);
    T* px = a.v_x ? static_cast<T*>(a.v_x) + (p.chain * a.chain_rows + p_first) * a.h_stride + p.channel : nullptr;
    const long long gate_row = (p.chain * a.chain_rows + p_first);
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
        const int s = first_at<TABLE>(p, first, l), e = end_at<TABLE>(p, end, l);
        if (e >= 0 && p.active) load_state<V>(a.v_state_out, e, a.channels, p.channel, q);
        const bool row_there = p_first + l < a.chain_rows;
        float dx[V], dg[V], sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool outside = s == kOutside || !p.active;
            const float f = s == kOutside ? 1.f : gate_f(m[l][v], a.logit), k = gate_k(m[l][v], a.logit);
            const float g = d[l][v] + q[v];
            dx[v] = outside ? 0.f : a.coupled ? k * g : g;
            dg[v] = outside ? 0.f : a.logit ? g * u[l][v] * (f * k) : g * u[l][v];
            sum += dg[v];
            q[v] = f * g;
        }
        if (px && p.active && row_there) store_floats<T, V>(px + l * a.h_stride, dx);
        if (s >= 0 && p.active && a.v_state_in) store_floats<float, V>(a.v_state_in + (long long)s * a.channels + p.channel, q);
        if (a.v_gate) {
            if (!a.shared) {
                if (p.active && row_there) store_floats<T, V>(static_cast<T*>(a.v_gate) + (gate_row + l) * a.gate_out_stride + p.channel, dg);
            } else {
                for (int off = (1 << a.lg_tx) >> 1; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (p.tx == 0 && row_there) {
                    const long long o = (gate_row + l) * a.gate_out_stride + p.head;
                    if (a.parts == 1) from_float(sum, static_cast<T*>(a.v_gate)[o]);
                    else a.gate_parts[(a.reverse ? (a.rows - 1) * a.gate_heads + o : o) + (long long)p.part * a.rows * a.gate_heads] = sum;
                }
            }
        }
    }
    pass_empty_sequences(a, a.v_state_out, a.v_state_in);
}

// v_gate = sum of the channel blocks' shares of it, in their order
template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_gate_sum_kernel(const float* parts, int count, long long n, T* v_gate) {
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kThreads) {
        float sum = 0.f;
        for (int k = 0; k < count; ++k) sum += parts[k * n + i];
        from_float(sum, v_gate[i]);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
recurrence_step_kernel(const T* x, const T* gate, float* state, T* h, const long long count, const int channels, const int per_head,
                       const long long x_stride, const long long gate_stride, const int logit, const int coupled, const int shared) {
    const long long i = ((long long)blockIdx.x * kThreads + threadIdx.x) * V;
    if (i >= count) return;
    const long long s = i / channels;
    const int c = (int)(i - s * channels);
    const Pack<T, V> px = load_pack<T, V>(x + s * x_stride + c);
    const Pack<float, V> ps = load_pack<float, V>(state + i);
    Pack<T, V> pg;
    if (shared) pg.e[0] = gate[s * gate_stride + c / per_head];
    else pg = load_pack<T, V>(gate + s * gate_stride + c);
    float o[V], m0 = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float m = shared && v > 0 ? m0 : encode_gate(to_float(pg.e[v]), logit);
        m0 = m;
        const float xv = to_float(px.e[v]);
        o[v] = fmaf(gate_f(m, logit), ps.e[v], coupled ? gate_k(m, logit) * xv : xv);
    }
    store_floats<float, V>(state + i, o);
    store_floats<T, V>(h + i, o);
}

// ---- host ----------------------------------------------------------------------------------------------------------------

constexpr int rows_per_thread(int vec, bool forward) { return vec == 4 ? (forward ? 8 : 4) : (forward ? 16 : 8); }
int tile_rows_of(const Layout& l, bool forward) { return kWarps * (32 >> l.lg_tx) * rows_per_thread(l.vec, forward); }

int check_shape(const DsbRecurrence& s, bool step) {
    DSB_REQUIRE(s.dtype == DSB_DTYPE_F32 || s.dtype == DSB_DTYPE_F16 || s.dtype == DSB_DTYPE_BF16, "recurrence: unknown dtype %d", s.dtype);
    DSB_REQUIRE(s.gate_form == DSB_GATE_DECAY || s.gate_form == DSB_GATE_LOGIT, "recurrence: unknown gate form %d", s.gate_form);
    DSB_REQUIRE(s.channels >= 1 && s.gate_heads >= 1 && s.channels % s.gate_heads == 0,
                "recurrence: %d channels do not split into %d gate heads", s.channels, s.gate_heads);
    DSB_REQUIRE(s.rows >= 0 && s.rows <= kMaxRows, "recurrence: at most 2^31 - 1 rows, got %lld", (long long)s.rows);
    DSB_REQUIRE(s.sequences >= 0, "recurrence: negative number of sequences");
    if (step) {
        DSB_REQUIRE(s.rows == s.sequences, "recurrence: a step takes one row per sequence");
        return DSB_OK;
    }
    DSB_REQUIRE(s.sequence_rows >= 0, "recurrence: negative sequence_rows");
    if (s.sequence_rows > 0) {
        DSB_REQUIRE((int64_t)s.sequences * s.sequence_rows == s.rows, "recurrence: %d sequences of %d rows are not %lld rows",
                    s.sequences, s.sequence_rows, (long long)s.rows);
        DSB_REQUIRE(!s.offsets, "recurrence: offsets are for packed rows (sequence_rows == 0)");
    } else {
        DSB_REQUIRE(!s.lengths, "recurrence: lengths are for sequences of sequence_rows rows");
        DSB_REQUIRE(s.offsets || s.rows == 0, "recurrence: packed rows need offsets");
    }
    return DSB_OK;
}

// The cut depends on the shape alone, never on addresses: the checkpoints of a forward fit every backward of the shape.
Layout layout_of(const DsbRecurrence& s, int vec) {
    Layout l;
    l.vec = vec;
    const bool shared = s.gate_heads != s.channels;
    l.heads = shared ? s.gate_heads : 1;
    l.per_head = s.channels / l.heads;
    const int wide = (l.per_head + l.vec - 1) / l.vec;
    l.lg_tx = 0;
    while (l.lg_tx < 5 && (1 << l.lg_tx) < wide) ++l.lg_tx;
    l.parts = (wide + (1 << l.lg_tx) - 1) >> l.lg_tx;
    // A chain per sequence wastes half a tile per sequence on average; a table costs a look at every row.
    l.table = s.sequence_rows == 0 || s.sequence_rows < tile_rows_of(l, true);
    l.chains = l.table ? 1 : s.sequences;
    l.chain_rows = l.table ? s.rows : s.sequence_rows;
    return l;
}
int shape_vec(const DsbRecurrence& s) {
    const bool shared = s.gate_heads != s.channels;
    return (shared ? s.channels / s.gate_heads : s.channels) % 4 == 0 ? 4 : 1;
}
int64_t chunks_of(const Layout& l, bool forward) {
    const int t = tile_rows_of(l, forward);
    return (l.chain_rows + t - 1) / t;
}
int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }

int64_t direction_workspace(const DsbRecurrence& s, const Layout& l, bool forward) {
    const int64_t maps = l.chains * chunks_of(l, forward);
    int64_t bytes = 0;
    if (chunks_of(l, forward) > 1) bytes += 2 * up16(maps * s.channels * 4) + up16(maps * 4);
    if (!forward && s.gate_heads != s.channels && l.parts > 1) bytes += up16((int64_t)l.parts * s.rows * s.gate_heads * 4);
    return bytes;
}

bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

struct Cut { Layout layout; Args args; int64_t tiles; };

int make_cut(const DsbRecurrence& s, bool forward, void* workspace, int64_t workspace_bytes, float* checkpoints, Cut* out) {
    Cut& c = *out;
    const int vec = shape_vec(s);
    c.layout = layout_of(s, vec);
    const Layout& l = c.layout;
    const int64_t need = direction_workspace(s, l, forward);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        set_error("recurrence: workspace of %lld bytes, %lld needed", (long long)(workspace ? workspace_bytes : 0), (long long)need);
        return DSB_ERR_WORKSPACE_TOO_SMALL;
    }
    DSB_REQUIRE(aligned(workspace, 16) && aligned(checkpoints, 16), "recurrence: workspace and checkpoints must be 16-byte aligned");
    Args& a = c.args;
    a = Args{};
    a.rows = s.rows; a.chain_rows = l.chain_rows; a.chains = l.chains;
    a.chunks = chunks_of(l, forward);
    a.checkpoint_rows = tile_rows_of(l, false); a.checkpoint_chunks = chunks_of(l, false);
    a.checkpoints = checkpoints;
    a.sequences = s.sequences; a.sequence_rows = s.sequence_rows; a.channels = s.channels; a.gate_heads = s.gate_heads;
    a.heads = l.heads; a.per_head = l.per_head; a.parts = l.parts; a.lg_tx = l.lg_tx;
    a.logit = s.gate_form == DSB_GATE_LOGIT; a.coupled = s.coupled != 0; a.reverse = s.reverse != 0;
    a.shared = s.gate_heads != s.channels;
    a.offsets = s.offsets; a.lengths = s.lengths;
    const int64_t sign = a.reverse ? -1 : 1;
    a.x_stride = sign * s.x_stride; a.gate_stride = sign * s.gate_stride;
    a.h_stride = sign * s.channels; a.gate_out_stride = sign * s.gate_heads;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    if (a.chunks > 1) {
        const int64_t maps = l.chains * a.chunks, bytes = up16(maps * s.channels * 4);
        a.map_a = reinterpret_cast<float*>(w); w += bytes;
        a.map_b = reinterpret_cast<float*>(w); w += bytes;
        a.map_closed = reinterpret_cast<int*>(w); w += up16(maps * 4);
    }
    if (!forward && a.shared && l.parts > 1) a.gate_parts = reinterpret_cast<float*>(w);
    c.tiles = l.chains * a.chunks * l.heads * l.parts;
    DSB_REQUIRE(c.tiles <= kMaxRows, "recurrence: too many tiles for one launch");
    return device_status_address(&a.device_status);
}

// Row r of the scan is row rows - 1 - r of the tensor when the scan runs backwards.
template <typename T>
T* scan_base(T* base, bool reverse, int64_t rows, int64_t stride, int elem) {
    if (!base || !reverse || rows == 0) return base;
    typedef typename std::conditional<std::is_const<T>::value, const char, char>::type Byte;
    return reinterpret_cast<T*>(reinterpret_cast<Byte*>(base) + (rows - 1) * stride * elem);
}

// No rows: nothing to scan, the states pass.
int pass_states(const float* in, float* out, int64_t count, cudaStream_t s) {
    if (!out || count == 0 || in == out) return DSB_OK;
    if (in) DSB_CUDA_CHECK(cudaMemcpyAsync(out, in, count * 4, cudaMemcpyDeviceToDevice, s));
    else DSB_CUDA_CHECK(cudaMemsetAsync(out, 0, count * 4, s));
    return DSB_OK;
}

template <typename T, int V, bool FORWARD>
int run_tiles(const Cut& c, cudaStream_t s) {
    const Args& a = c.args;
    const bool table = c.layout.table;
    constexpr int L = rows_per_thread(V, FORWARD);
    const size_t smem = table ? 2 * sizeof(int) * tile_rows_of(c.layout, FORWARD) : 0;
    const unsigned grid = (unsigned)c.tiles;
    auto launch = [&](auto apply) {
        constexpr bool APPLY = decltype(apply)::value;
        if (FORWARD) {
            if (table) recurrence_forward_kernel<T, V, L, true, APPLY><<<grid, kThreads, smem, s>>>(a);
            else recurrence_forward_kernel<T, V, L, false, APPLY><<<grid, kThreads, smem, s>>>(a);
        } else {
            if (table) recurrence_backward_kernel<T, V, L, true, APPLY><<<grid, kThreads, smem, s>>>(a);
            else recurrence_backward_kernel<T, V, L, false, APPLY><<<grid, kThreads, smem, s>>>(a);
        }
    };
    if (a.chunks > 1) {
        launch(std::false_type{});
        DSB_LAUNCH_CHECK();
        const unsigned carry_grid = (unsigned)((a.chains * a.channels + kThreads - 1) / kThreads);
        recurrence_carry_kernel<FORWARD><<<carry_grid, kThreads, 0, s>>>(a);
        DSB_LAUNCH_CHECK();
    }
    launch(std::true_type{});
    DSB_LAUNCH_CHECK();
    return DSB_OK;
}

template <bool FORWARD>
int run_direction(const DsbRecurrence& shape, const Cut& c, cudaStream_t s) {
    int rc = DSB_OK;
    with_dtype(shape.dtype, [&](auto tag) {
        typedef decltype(tag) T;
        rc = c.layout.vec == 4 ? run_tiles<T, 4, FORWARD>(c, s) : run_tiles<T, 1, FORWARD>(c, s);
        if (rc == DSB_OK && !FORWARD && c.args.gate_parts && c.args.v_gate) {
            const long long n = shape.rows * shape.gate_heads;
            T* out = static_cast<T*>(c.args.v_gate);
            if (c.args.reverse) out -= (shape.rows - 1) * shape.gate_heads;
            const long long blocks = (n + kThreads - 1) / kThreads;
            recurrence_gate_sum_kernel<T><<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), kThreads, 0, s>>>(
                c.args.gate_parts, c.layout.parts, n, out);
            count_launch();
            if (cudaPeekAtLastError() != cudaSuccess) { set_error("recurrence: launch failed"); rc = DSB_ERR_CUDA; }
        }
    });
    return rc;
}

// Vector tiles (four channels a thread) need every row of every tensor on a boundary of four elements.
int check_alignment(const DsbRecurrence& s, const void* p, int64_t stride, int elem, bool wide, const char* name) {
    if (!p || !wide) return DSB_OK;
    DSB_REQUIRE(aligned(p, 4 * elem) && stride % 4 == 0,
                "recurrence: with channels in fours, %s must start on a boundary of four elements and its rows lie a multiple of "
                "four elements apart", name);
    return DSB_OK;
}
#define DSB_TRY(expr) do { const int rc__ = (expr); if (rc__ != DSB_OK) return rc__; } while (0)

int check_inputs(const DsbRecurrence& s, const void* x, const void* gate) {
    const bool wide = shape_vec(s) == 4;
    const int elem = dtype_bytes(s.dtype);
    DSB_TRY(check_alignment(s, x, s.x_stride, elem, wide, "x"));
    return check_alignment(s, gate, s.gate_stride, elem, wide && s.gate_heads == s.channels, "the gate");
}

}  // namespace

int64_t recurrence_workspace_bytes(const DsbRecurrence& s) {
    if (check_shape(s, false) != DSB_OK) return 0;
    const Layout l = layout_of(s, shape_vec(s));
    const int64_t f = direction_workspace(s, l, true), b = direction_workspace(s, l, false);
    return f > b ? f : b;
}

int64_t recurrence_checkpoint_bytes(const DsbRecurrence& s) {
    if (check_shape(s, false) != DSB_OK) return 0;
    const Layout l = layout_of(s, shape_vec(s));
    return l.chains * chunks_of(l, false) * s.channels * 4;
}

int launch_recurrence_forward(const DsbRecurrence& shape, const void* x, const void* gate, const float* state_in, void* h,
                              float* state_out, float* checkpoints, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
    DSB_TRY(check_shape(shape, false));
    DSB_REQUIRE(state_out || shape.sequences == 0, "recurrence: null state_out");
    if (shape.rows == 0) return pass_states(state_in, state_out, (int64_t)shape.sequences * shape.channels, s);
    DSB_REQUIRE(x && gate, "recurrence: null pointer");
    DSB_REQUIRE(!state_in || state_in != state_out, "recurrence: state_out must not be state_in");
    const bool wide = shape_vec(shape) == 4;
    const int elem = dtype_bytes(shape.dtype);
    DSB_TRY(check_inputs(shape, x, gate));
    DSB_TRY(check_alignment(shape, h, shape.channels, elem, wide, "h"));
    DSB_TRY(check_alignment(shape, state_in, shape.channels, 4, wide, "state_in"));
    DSB_TRY(check_alignment(shape, state_out, shape.channels, 4, wide, "state_out"));
    Cut c;
    DSB_TRY(make_cut(shape, true, workspace, workspace_bytes, checkpoints, &c));
    const bool r = shape.reverse != 0;
    c.args.x = scan_base(x, r, shape.rows, shape.x_stride, elem);
    c.args.gate = scan_base(gate, r, shape.rows, shape.gate_stride, elem);
    c.args.h = scan_base(h, r, shape.rows, shape.channels, elem);
    c.args.state_in = state_in; c.args.state_out = state_out;
    return run_direction<true>(shape, c, s);
}

int launch_recurrence_backward(const DsbRecurrence& shape, const void* x, const void* gate, const float* state_in,
                               const float* checkpoints, const void* v_h, int64_t v_h_stride, const float* v_state_out,
                               void* v_x, void* v_gate, float* v_state_in, void* workspace, int64_t workspace_bytes,
                               cudaStream_t s) {
    DSB_TRY(check_shape(shape, false));
    if (shape.rows == 0) return pass_states(v_state_out, v_state_in, (int64_t)shape.sequences * shape.channels, s);
    DSB_REQUIRE(x && gate && checkpoints, "recurrence: null pointer");
    DSB_REQUIRE(!v_state_in || v_state_in != v_state_out, "recurrence: v_state_in must not be v_state_out");
    const bool wide = shape_vec(shape) == 4;
    const int elem = dtype_bytes(shape.dtype);
    DSB_TRY(check_inputs(shape, x, gate));
    DSB_TRY(check_alignment(shape, v_h, v_h_stride, elem, wide, "v_h"));
    DSB_TRY(check_alignment(shape, v_x, shape.channels, elem, wide, "v_x"));
    DSB_TRY(check_alignment(shape, v_gate, shape.gate_heads, elem, wide && shape.gate_heads == shape.channels, "v_gate"));
    DSB_TRY(check_alignment(shape, state_in, shape.channels, 4, wide, "state_in"));
    DSB_TRY(check_alignment(shape, v_state_out, shape.channels, 4, wide, "v_state_out"));
    DSB_TRY(check_alignment(shape, v_state_in, shape.channels, 4, wide, "v_state_in"));
    Cut c;
    DSB_TRY(make_cut(shape, false, workspace, workspace_bytes, const_cast<float*>(checkpoints), &c));
    const bool r = shape.reverse != 0;
    c.args.x = scan_base(x, r, shape.rows, shape.x_stride, elem);
    c.args.gate = scan_base(gate, r, shape.rows, shape.gate_stride, elem);
    c.args.v_h = scan_base(v_h, r, shape.rows, v_h_stride, elem);
    c.args.v_h_stride = r ? -v_h_stride : v_h_stride;
    c.args.v_x = scan_base(v_x, r, shape.rows, shape.channels, elem);
    c.args.v_gate = scan_base(v_gate, r, shape.rows, shape.gate_heads, elem);
    c.args.state_in = state_in; c.args.v_state_out = v_state_out; c.args.v_state_in = v_state_in;
    return run_direction<false>(shape, c, s);
}

int launch_recurrence_step(const DsbRecurrence& shape, const void* x, const void* gate, float* state, void* h, cudaStream_t s) {
    DSB_TRY(check_shape(shape, true));
    if (shape.rows == 0) return DSB_OK;
    DSB_REQUIRE(x && gate && state && h, "recurrence: null pointer");
    const bool wide = shape_vec(shape) == 4;
    const int elem = dtype_bytes(shape.dtype);
    DSB_TRY(check_inputs(shape, x, gate));
    DSB_TRY(check_alignment(shape, h, shape.channels, elem, wide, "h"));
    DSB_TRY(check_alignment(shape, state, shape.channels, 4, wide, "the state"));
    const long long count = shape.rows * shape.channels;
    const long long blocks = (count / (wide ? 4 : 1) + kThreads - 1) / kThreads;
    DSB_REQUIRE(blocks <= kMaxRows, "recurrence: too many elements for one launch");
    const int per_head = shape.channels / shape.gate_heads, shared = per_head > 1;
    with_dtype(shape.dtype, [&](auto tag) {
        typedef decltype(tag) T;
        const T* tx = static_cast<const T*>(x);
        const T* tg = static_cast<const T*>(gate);
        T* th = static_cast<T*>(h);
        if (wide)
            recurrence_step_kernel<T, 4><<<(unsigned)blocks, kThreads, 0, s>>>(
                tx, tg, state, th, count, shape.channels, per_head, shape.x_stride, shape.gate_stride,
                shape.gate_form == DSB_GATE_LOGIT, shape.coupled != 0, shared);
        else
            recurrence_step_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, s>>>(
                tx, tg, state, th, count, shape.channels, per_head, shape.x_stride, shape.gate_stride,
                shape.gate_form == DSB_GATE_LOGIT, shape.coupled != 0, shared);
    });
    DSB_LAUNCH_CHECK();
    return DSB_OK;
}

}  // namespace dsb
