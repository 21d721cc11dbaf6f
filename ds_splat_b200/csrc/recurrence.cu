// Gated linear recurrence over sequences, forward and backward, and its single-row form:
//     f_t = gate_t or 1 / (1 + exp(-gate_t)),   h_t = f_t h_{t-1} + i_t,   i_t = x_t or, coupled, (1 - f_t) x_t
//     g_t = v_h_t + q_{t+1},   q_t = f_t g_t,   v_x_t = g_t or (1 - f_t) g_t
//     v_f_t = sum over the channels that share the gate of g_t (h_{t-1}, coupled: h_{t-1} - x_t),   v_state_in = q_0
// Not part of the reference as an operator of its own; its blend (cpp/rasterizer_kernels.cu:341-431) is the coupled form
// over a tile's list, back to front, with f = 1 - alpha.
//
// A stretch of rows maps the state before it to the state after it as h -> a h + b, and two stretches compose as
// (a2 a1, a2 b1 + b2); a stretch in which a sequence begins maps every h to b ("closed": its a is never looked at, so
// that an infinity of the sequence before cannot meet a zero).
//
// A block walks along one stretch of rows and a block of channels, tile by tile, and carries the state in registers: it
// reads everything once and writes everything once.  Inside a tile a thread runs L consecutive rows of V channels, a warp
// composes its threads' maps with shuffles, the block its warps' through shared memory (one barrier a tile); the next
// tile's rows are on their way into shared memory meanwhile (each thread copies what it will read itself, so their arrival
// needs no barrier).  Where sequences and channels alone make too few blocks for the GPU, a sequence is cut into segments:
// a first launch leaves every segment's map, and each block of the second starts from the composition of those before it.
// That reads the inputs twice, the second time mostly from L2 where the call is small enough to need it.
//
// The backward walks from the last row to the first on q, and recomputes h inside a tile from the state the tile starts
// with (a checkpoint of the forward), in 32 bits: the h that was written out is rounded to the storage type and need not
// be kept.  Every order of composition is fixed by the shape alone, so results do not depend on timing; no block waits for
// another.
#include <type_traits>

#include "vector_io.cuh"

namespace dsb {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr long long kMaxRows = (1ll << 31) - 1;
constexpr int kStages = 2;
constexpr int kTables = 3;      // one is read, one was read by the slowest warp, one is written

struct Layout {            // how a call is cut; the same for the forward and the backward of one shape
    int vec;               // channels per thread: 4 or 1
    int lg_tx;             // log2 of the threads side by side on one row
    int per_head;          // channels that share a gate; all of them when every channel has its own
    int heads;             // 1 when every channel has its own gate
    int parts;             // channel blocks per head
    bool table;            // tiles may hold sequence borders: one chain over all rows; else one chain per sequence
    int tile_rows;
    long long chains, chain_rows, tiles;   // tiles of a chain
    long long segments, segment_tiles;     // of a chain
};

struct Args {
    const void *x, *gate, *v_h;
    void *h, *v_x, *v_gate;
    const float *state_in, *v_state_out;
    float *state_out, *v_state_in;
    float* checkpoints;    // [chains][tiles][channels]: the state before each tile
    float *map_a, *map_b;  // [chains][segments][channels]
    int* map_closed;       // [chains][segments]
    float* gate_parts;     // [parts][rows][heads], when a head spans several channel blocks
    const int *offsets, *lengths;
    int* device_status;
    long long rows, chain_rows, chains;
    long long x_stride, gate_stride, v_h_stride;   // negative when the scan runs from the last row to the first
    long long h_stride, gate_out_stride;           // channels / heads of contiguous results, with the same sign
    long long tiles, segments, segment_tiles;
    int sequences, sequence_rows, channels, gate_heads, heads, per_head, parts, lg_tx;
    int logit, coupled, reverse, shared;
};

// ---- gates ---------------------------------------------------------------------------------------------------------
// One register holds both f and 1 - f to full relative precision where they are small: for a logit the smaller of the two,
// m = exp(-|g|) / (1 + exp(-|g|)) <= 1/2, with the sign saying which one it is.
__device__ __forceinline__ float encode_gate(float g, int logit) {
    if (!logit) return g;
    float y, r;
    asm("max.NaN.f32 %0, %1, 0fC2B40000;" : "=f"(y) : "f"(-fabsf(g)));   // -90: exp is 0 beside 1 long before; NaN stays NaN
    // exp(y) = 2^(y log2 e), the product's rounding error added back to first order
    const float hi = y * 1.44269502f;
    const float lo = fmaf(y, 1.44269502f, -hi);
    float t = exp2f(hi);
    t = fmaf(t, lo * 0.693147181f, t);
    t = y <= -90.f ? 0.f : t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + t));
    return copysignf(t * r, g);
}
__device__ __forceinline__ void decode_gate(float m, int logit, float& f, float& k) {
    const float rest = 1.f - (logit ? fabsf(m) : m);
    const bool small_f = logit ? __float_as_int(m) < 0 : true;   // a decay is f itself
    const float own = logit ? fabsf(m) : m;
    f = small_f ? own : rest;
    k = small_f ? rest : own;
}

// ---- rows that begin and end sequences ------------------------------------------------------------------------------
// In the order of the scan: position p is row p, or rows - 1 - p when the scan runs backwards; sequence k of the scan is
// the tensor's sequence k, or sequences - 1 - k.
constexpr int kNone = -1, kOutside = -2;

__device__ __forceinline__ int sequence_id(const Args& a, int k) { return a.reverse ? a.sequences - 1 - k : k; }
// Where the scan's packed sequence k begins (k = sequences: where the last one ends).
__device__ __forceinline__ long long packed_start(const Args& a, long long k) {
    return a.reverse ? a.rows - a.offsets[a.sequences - k] : a.offsets[k];
}
struct ChainRows {         // without a table: the chain is one sequence, and holds positions [lo, hi)
    int sequence;
    long long lo, hi;
};
__device__ __forceinline__ ChainRows chain_rows_of(const Args& a, int chain) {
    ChainRows c;
    c.sequence = sequence_id(a, chain);
    long long len = a.sequence_rows;
    if (a.lengths) len = min(max(a.lengths[c.sequence], 0), a.sequence_rows);
    c.lo = a.reverse ? a.sequence_rows - len : 0;
    c.hi = c.lo + len;
    return c;
}

// How many of the scan's packed sequences k begin at or before p; called by one whole warp.
__device__ __forceinline__ int begun_by(const Args& a, long long p) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = a.sequences;
    while (len > 0) {
        const int step = (len + 31) / 32;
        const long long at = (long long)lane * step;
        const bool below = at < len && packed_start(a, lo + at) <= p;
        const int below_count = __popc(__ballot_sync(0xffffffffu, below));
        if (below_count == 0) break;
        const int skip = (below_count - 1) * step + 1;
        len = min(step - 1, len - skip);
        lo += skip;
    }
    return lo;
}

// first[r] / end[r]: the sequence that begins / ends at position p0 + r, kNone, or (first only) kOutside.  A tile is plain
// when all its rows belong to a sequence that neither begins nor ends there.  Tables are made for one tile while the one
// before it is worked on; the block's next barrier publishes them.  `cursor` is the scan's sequence to begin looking at (the
// last to begin at or before p0); in shared memory, kept by this function from tile to tile.
struct RowTable {
    int* first;
    int* end;
};
__device__ void fill_row_table(const Args& a, long long p0, int tile_rows, RowTable t) {
    const int tid = threadIdx.x;
    if (a.sequence_rows > 0) {
        for (int r = tid; r < tile_rows; r += kThreads) {
            const long long p = p0 + r;
            int f = kOutside, e = kNone;
            if (p < a.rows) {
                const int turn = (int)(p / a.sequence_rows), pos = (int)(p - (long long)turn * a.sequence_rows);
                const int seq = sequence_id(a, turn);
                const int len = a.lengths ? min(max(a.lengths[seq], 0), a.sequence_rows) : a.sequence_rows;
                const int lo = a.reverse ? a.sequence_rows - len : 0;
                if (pos >= lo && pos < lo + len) {
                    f = pos == lo ? seq : kNone;
                    e = pos == lo + len - 1 ? seq : kNone;
                }
            }
            t.first[r] = f;
            t.end[r] = e;
        }
        return;
    }
    const long long p1 = min(p0 + tile_rows, a.rows);
    const long long all0 = packed_start(a, 0), all1 = packed_start(a, a.sequences);
    for (int r = tid; r < tile_rows; r += kThreads) {
        const long long p = p0 + r;
        t.first[r] = p < p1 && p >= all0 && p < all1 ? kNone : kOutside;
        t.end[r] = kNone;
    }
    int k0 = 0;
    if (tid < 32) k0 = max(begun_by(a, p0) - 1, 0);
    __shared__ int s_k0;
    if (tid == 0) s_k0 = k0;
    __syncthreads();
    for (long long k = s_k0 + tid; k < a.sequences; k += kThreads) {
        const long long o0 = packed_start(a, k), o1 = packed_start(a, k + 1);
        if (o0 >= p1) break;
        if (o0 >= o1) continue;
        const int id = sequence_id(a, (int)k);
        if (o0 >= p0) t.first[o0 - p0] = id;
        if (o1 > p0 && o1 <= p1) t.end[o1 - 1 - p0] = id;
    }
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
    const bool open = !m.closed;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        m.b[v] = open ? fmaf(m.a[v], e.b[v], m.b[v]) : m.b[v];
        m.a[v] *= e.a[v];
    }
    m.closed |= e.closed;
}
template <int V>
__device__ __forceinline__ void apply_map(float (&h)[V], const Map<V>& m) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = m.closed ? m.b[v] : fmaf(m.a[v], h[v], m.b[v]);
}

// The warps' maps of one tile, for one direction.
template <int V>
struct alignas(16) WarpMaps {     // read and written V floats at a time
    float a[kWarps][32 * V], b[kWarps][32 * V];
    int closed[kWarps];
};

// Lanes that hold the same channels on consecutive row groups are tx apart.  From every thread's own map: the warp's
// total in shared memory, and the map of the warp's rows before this thread's.  FORWARD: rows run with the lane; else
// against it.
template <int V, bool FORWARD>
__device__ __forceinline__ Map<V> compose_warp(const Map<V>& own, int lg_tx, WarpMaps<V>& sh) {
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
        store_floats<float, V>(&sh.a[warp][at], run.a);
        store_floats<float, V>(&sh.b[warp][at], run.b);
        if ((lane & (tx - 1)) == 0) sh.closed[warp] = run.closed;
    }
    Map<V> before;
    identity(before);
    if (tx < 32) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            before.a[v] = FORWARD ? __shfl_up_sync(0xffffffffu, run.a[v], tx) : __shfl_down_sync(0xffffffffu, run.a[v], tx);
            before.b[v] = FORWARD ? __shfl_up_sync(0xffffffffu, run.b[v], tx) : __shfl_down_sync(0xffffffffu, run.b[v], tx);
        }
        before.closed = FORWARD ? __shfl_up_sync(0xffffffffu, run.closed, tx) : __shfl_down_sync(0xffffffffu, run.closed, tx);
        if (FORWARD ? lane < tx : lane >= 32 - tx) identity(before);
    }
    return before;
}
template <int V>
__device__ __forceinline__ Map<V> warp_map(const WarpMaps<V>& sh, int warp, int tx) {
    Map<V> m;
    const Pack<float, V> pa = load_pack<float, V>(&sh.a[warp][tx * V]), pb = load_pack<float, V>(&sh.b[warp][tx * V]);
#pragma unroll
    for (int v = 0; v < V; ++v) { m.a[v] = pa.e[v]; m.b[v] = pb.e[v]; }
    m.closed = sh.closed[warp];
    return m;
}
// carry: the state before the tile -> the state after it.  Returns the state before this thread's warp.
template <int V, bool FORWARD>
__device__ __forceinline__ void pass_warps(const WarpMaps<V>& sh, int tx, float (&carry)[V], float (&mine)[V]) {
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const int w = FORWARD ? i : kWarps - 1 - i;
        if (w == warp) {
#pragma unroll
            for (int v = 0; v < V; ++v) mine[v] = carry[v];
        }
        apply_map(carry, warp_map<V>(sh, w, tx));
    }
}

// ---- a block's place -----------------------------------------------------------------------------------------------------
struct Place {
    int chain, head, part, channel, tx;
    long long segment;
    int row0;              // this thread's first row inside a tile
    bool active;
    ChainRows rows;
};
template <int V, int L, bool TABLE>
__device__ __forceinline__ Place place_of(const Args& a) {
    Place p;
    const int blocks = a.heads * a.parts;
    const long long rest = blockIdx.x / blocks;
    const int block = (int)(blockIdx.x - rest * blocks);
    p.chain = (int)(rest % a.chains);
    p.segment = rest / a.chains;
    p.head = block / a.parts;
    p.part = block - p.head * a.parts;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    p.tx = lane & ((1 << a.lg_tx) - 1);
    p.row0 = (warp * (32 >> a.lg_tx) + (lane >> a.lg_tx)) * L;
    const int c = (p.part << a.lg_tx) * V + p.tx * V;
    p.active = c < a.per_head;
    p.channel = p.head * a.per_head + c;
    if (!TABLE) p.rows = chain_rows_of(a, p.chain);
    return p;
}

// What a thread knows of its L rows of one tile.  first(l) / end(l): the sequence that begins / ends there, or negative.
template <int L, bool TABLE>
struct Rows {
    const int *t_first, *t_end;
    int lo, hi, sequence;      // without a table: rows l in [lo, hi) belong to `sequence`, which begins at lo and ends at hi - 1
    __device__ __forceinline__ Rows(const Place& p, long long p0, RowTable t) {
        if (TABLE) {
            t_first = t.first + p.row0;
            t_end = t.end + p.row0;
        } else {
            const long long at = p0 + p.row0;
            lo = (int)min(max(p.rows.lo - at, -1ll), (long long)L);       // -1: began before
            hi = (int)min(max(p.rows.hi - at, -1ll), (long long)L + 1);   // L + 1: goes on
            sequence = p.rows.sequence;
        }
    }
    __device__ __forceinline__ bool outside(int l) const { return TABLE ? t_first[l] == kOutside : l < lo || l >= hi; }
    __device__ __forceinline__ int first(int l) const { return TABLE ? t_first[l] : l == lo && l < hi ? sequence : kNone; }
    __device__ __forceinline__ int end(int l) const { return TABLE ? t_end[l] : l == hi - 1 && l >= lo ? sequence : kNone; }
};

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

// ---- rows on their way through shared memory ---------------------------------------------------------------------------
// A thread's V elements of row l, tensor k: slot (k L + l) of the stage, lanes side by side.
template <typename T, int V>
__device__ __forceinline__ void copy_async(T* to, const T* from, bool there) {
    constexpr int kBytes = V * sizeof(T);
    if (kBytes == 2) {
        memset(to, 0, kBytes);
        if (there) *to = *from;
    } else {
        const unsigned at = (unsigned)__cvta_generic_to_shared(to);
        const int bytes = there ? kBytes : 0;    // what is not copied is filled with zeros
        if (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
        else if (kBytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
    }
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <typename T, int V, int L, int TENSORS>
struct alignas(16) Stage {
    T v[TENSORS][L][kThreads][V];
};

// Rows p0 + row0 .. of one tensor; rows past the chain's end become zeros.  Rows that belong to no sequence but lie within
// the tensor are copied like the others and masked where they are used.
template <typename T, int V, int L>
__device__ __forceinline__ void fetch_rows(T (*to)[kThreads][V], const T* base, long long stride, const Args& a, const Place& p,
                                           long long p0) {
    const long long at = p0 + p.row0;
    const T* from = base + (p.chain * a.chain_rows + at) * stride;
    const int left = p.active ? (int)min(a.chain_rows - at, (long long)L) : 0;
#pragma unroll
    for (int l = 0; l < L; ++l) copy_async<T, V>(to[l][threadIdx.x], l < left ? from + l * stride : base, l < left);
}
// The gates of the rows, encoded.  Shared ones are read directly: every thread of a row wants the same value.
template <typename T, int V, int L>
__device__ __forceinline__ void fetch_gates(T (*to)[kThreads][V], T (&own)[L], const Args& a, const Place& p, long long p0) {
    const T* base = static_cast<const T*>(a.gate) + (a.shared ? p.head : p.channel);
    if (!a.shared) {
        fetch_rows<T, V, L>(to, base, a.gate_stride, a, p, p0);
        return;
    }
    const long long at = p0 + p.row0;
    const T* from = base + (p.chain * a.chain_rows + at) * a.gate_stride;
    const int left = p.active ? (int)min(a.chain_rows - at, (long long)L) : 0;
#pragma unroll
    for (int l = 0; l < L; ++l) {
        if (l < left) own[l] = from[l * a.gate_stride];
        else memset(&own[l], 0, sizeof(T));
    }
}
template <typename T, int V, int L>
__device__ __forceinline__ void read_gates(const T (*from)[kThreads][V], const T (&own)[L], const Args& a, float (&m)[L][V]) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
        if (a.shared) {
            const float one = encode_gate(to_float(own[l]), a.logit);
#pragma unroll
            for (int v = 0; v < V; ++v) m[l][v] = one;
        } else {
            const Pack<T, V> g = load_pack<T, V>(from[l][threadIdx.x]);
#pragma unroll
            for (int v = 0; v < V; ++v) m[l][v] = encode_gate(to_float(g.e[v]), a.logit);
        }
    }
}

// The state (or q) at the segment's beginning: the maps of the segments before it, each warp a share of them, in order.
template <int V, bool FORWARD>
__device__ void carry_of_segment(const Args& a, const Place& p, WarpMaps<V>& sh, float (&carry)[V]) {
    const long long before = FORWARD ? p.segment : a.segments - 1 - p.segment;
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = 0.f;
    if (before == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long share = (before + kWarps - 1) / kWarps;
    const long long i0 = min(share * warp, before), i1 = min(i0 + share, before);
    Map<V> all;
    identity(all);
    if (lane < (1 << a.lg_tx)) {
#pragma unroll 4
        for (long long i = i0; i < i1; ++i) {
            const long long at = p.chain * a.segments + (FORWARD ? i : a.segments - 1 - i);
            Map<V> m;
            identity(m);
            m.closed = a.map_closed[at];
            if (p.active) {
                const Pack<float, V> pa = load_pack<float, V>(a.map_a + at * a.channels + p.channel);
                const Pack<float, V> pb = load_pack<float, V>(a.map_b + at * a.channels + p.channel);
#pragma unroll
                for (int v = 0; v < V; ++v) { m.a[v] = pa.e[v]; m.b[v] = pb.e[v]; }
            }
            compose_after(m, all);
            all = m;
        }
        store_floats<float, V>(&sh.a[warp][p.tx * V], all.a);
        store_floats<float, V>(&sh.b[warp][p.tx * V], all.b);
        if (p.tx == 0) sh.closed[warp] = all.closed;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) apply_map(carry, warp_map<V>(sh, w, p.tx));
    __syncthreads();
}

// Leaves the composition of a whole segment's tiles (APPLY = false).
template <int V>
__device__ __forceinline__ void store_segment_map(const Args& a, const Place& p, const Map<V>& all) {
    if (threadIdx.x >= (1 << a.lg_tx) || !p.active) return;
    const long long at = p.chain * a.segments + p.segment;
    store_floats<float, V>(a.map_a + at * a.channels + p.channel, all.a);
    store_floats<float, V>(a.map_b + at * a.channels + p.channel, all.b);
    if (p.tx == 0) a.map_closed[at] = all.closed;
}

template <typename T, int V, int L, bool TABLE, bool APPLY>
__global__ void __launch_bounds__(kThreads)
recurrence_forward_kernel(const Args a) {
    typedef Stage<T, V, L, 2> Ring;
    extern __shared__ __align__(16) unsigned char s_raw[];
    Ring* ring = reinterpret_cast<Ring*>(s_raw);
    int* tables = reinterpret_cast<int*>(s_raw + kStages * sizeof(Ring));
    __shared__ WarpMaps<V> sh[2];
    const int tile_rows = kWarps * (32 >> a.lg_tx) * L;
    const Place p = place_of<V, L, TABLE>(a);
    const long long t0 = p.segment * a.segment_tiles, t1 = min(t0 + a.segment_tiles, a.tiles);
    const T* x = static_cast<const T*>(a.x) + p.channel;
    auto table = [&](long long t) { int* at = tables + (int)(t % kTables) * 2 * tile_rows; return RowTable{at, at + tile_rows}; };

    float carry[V];
    Map<V> all;
    identity(all);
    if (APPLY) carry_of_segment<V, true>(a, p, sh[0], carry);
    T gate_now[L], gate_next[L];
    fetch_rows<T, V, L>(ring[0].v[0], x, a.x_stride, a, p, t0 * tile_rows);
    fetch_gates<T, V, L>(ring[0].v[1], gate_next, a, p, t0 * tile_rows);
    copies_issued();
    if (TABLE) {
        fill_row_table(a, t0 * tile_rows, tile_rows, table(t0));
        __syncthreads();
    }
    for (long long t = t0; t < t1; ++t) {
        const int stage = (int)(t - t0) & 1;
        const long long p0 = t * tile_rows;
#pragma unroll
        for (int l = 0; l < L; ++l) gate_now[l] = gate_next[l];
        if (t + 1 < t1) {
            fetch_rows<T, V, L>(ring[stage ^ 1].v[0], x, a.x_stride, a, p, p0 + tile_rows);
            fetch_gates<T, V, L>(ring[stage ^ 1].v[1], gate_next, a, p, p0 + tile_rows);
        }
        copies_issued();
        copies_landed<1>();
        const Rows<L, TABLE> rows(p, p0, table(t));
        float f[L][V], b[L][V];
        read_gates<T, V, L>(ring[stage].v[1], gate_now, a, f);
        Map<V> own;
        identity(own);
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int s = rows.first(l);
            const bool outside = rows.outside(l);
            const Pack<T, V> px = load_pack<T, V>(ring[stage].v[0][l][threadIdx.x]);
            float st[V];
            if (s >= 0) {
                own.closed = 1;
                if (p.active) load_state<V>(a.state_in, s, a.channels, p.channel, st);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float k;
                decode_gate(f[l][v], a.logit, f[l][v], k);
                const float xv = to_float(px.e[v]);
                b[l][v] = outside ? 0.f : a.coupled ? xv * k : xv;
                f[l][v] = outside ? 1.f : f[l][v];
                own.b[v] = fmaf(f[l][v], s >= 0 && p.active ? st[v] : own.b[v], b[l][v]);
                own.a[v] *= f[l][v];
            }
        }
        const Map<V> before = compose_warp<V, true>(own, a.lg_tx, sh[stage]);
        if (TABLE && t + 1 < t1) fill_row_table(a, p0 + tile_rows, tile_rows, table(t + 1));
        __syncthreads();
        if (!APPLY) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                Map<V> m = warp_map<V>(sh[stage], w, p.tx);
                compose_after(m, all);
                all = m;
            }
            continue;
        }
        if (a.checkpoints && threadIdx.x < (1 << a.lg_tx) && p.active)
            store_floats<float, V>(a.checkpoints + (p.chain * a.tiles + t) * a.channels + p.channel, carry);
        float h[V];
        pass_warps<V, true>(sh[stage], p.tx, carry, h);
        apply_map(h, before);
        T* ph = a.h ? static_cast<T*>(a.h) + (p.chain * a.chain_rows + p0 + p.row0) * a.h_stride + p.channel : nullptr;
        const int left = p.active ? (int)min(a.chain_rows - p0 - p.row0, (long long)L) : 0;
#pragma unroll
        for (int l = 0; l < L; ++l) {
            const int s = rows.first(l), e = rows.end(l);
            if (s >= 0 && p.active) load_state<V>(a.state_in, s, a.channels, p.channel, h);
            const bool outside = rows.outside(l);
            float o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = fmaf(f[l][v], h[v], b[l][v]);
                o[v] = outside ? 0.f : h[v];
            }
            if (ph && l < left) store_floats<T, V>(ph + l * a.h_stride, o);
            if (e >= 0 && p.active) store_floats<float, V>(a.state_out + (long long)e * a.channels + p.channel, h);
        }
    }
    if (APPLY) pass_empty_sequences(a, a.state_in, a.state_out);
    else store_segment_map<V>(a, p, all);
}

template <typename T, int V, int L, bool TABLE, bool APPLY>
__global__ void __launch_bounds__(kThreads)
recurrence_backward_kernel(const Args a) {
    typedef Stage<T, V, L, 3> Ring;
    extern __shared__ __align__(16) unsigned char s_raw[];
    Ring* ring = reinterpret_cast<Ring*>(s_raw);
    int* tables = reinterpret_cast<int*>(s_raw + kStages * sizeof(Ring));
    __shared__ WarpMaps<V> sh[2], sh_forward[2];
    const int tile_rows = kWarps * (32 >> a.lg_tx) * L;
    const Place p = place_of<V, L, TABLE>(a);
    const long long t0 = p.segment * a.segment_tiles, t1 = min(t0 + a.segment_tiles, a.tiles);
    const T* x = static_cast<const T*>(a.x) + p.channel;
    const T* vh = static_cast<const T*>(a.v_h) + p.channel;
    auto table = [&](long long t) { int* at = tables + (int)(t % kTables) * 2 * tile_rows; return RowTable{at, at + tile_rows}; };

    float q_carry[V], start[V], start_next[V];
    Map<V> all;
    identity(all);
    if (APPLY) carry_of_segment<V, false>(a, p, sh[0], q_carry);
    T gate_now[L], gate_next[L];
    auto fetch = [&](int stage, long long t) {
        if (a.v_h) fetch_rows<T, V, L>(ring[stage].v[0], vh, a.v_h_stride, a, p, t * tile_rows);
        fetch_gates<T, V, L>(ring[stage].v[1], gate_next, a, p, t * tile_rows);
        if (APPLY) {
            fetch_rows<T, V, L>(ring[stage].v[2], x, a.x_stride, a, p, t * tile_rows);
            load_state<V>(p.active ? a.checkpoints : nullptr, p.chain * a.tiles + t, a.channels, p.channel, start_next);
        }
    };
    fetch((int)(t1 - 1 - t0) & 1, t1 - 1);
    copies_issued();
    if (TABLE) {
        fill_row_table(a, (t1 - 1) * tile_rows, tile_rows, table(t1 - 1));
        __syncthreads();
    }
    for (long long t = t1 - 1; t >= t0; --t) {
        const int stage = (int)(t - t0) & 1;
        const long long p0 = t * tile_rows;
#pragma unroll
        for (int l = 0; l < L; ++l) gate_now[l] = gate_next[l];
#pragma unroll
        for (int v = 0; v < V; ++v) start[v] = start_next[v];
        if (t > t0) fetch(stage ^ 1, t - 1);
        copies_issued();
        copies_landed<1>();
        const Rows<L, TABLE> rows(p, p0, table(t));
        float m[L][V], u[L][V];
        read_gates<T, V, L>(ring[stage].v[1], gate_now, a, m);
        Map<V> own, before;
        if (APPLY) {
            identity(own);
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const int s = rows.first(l);
                const bool outside = rows.outside(l);
                const Pack<T, V> px = load_pack<T, V>(ring[stage].v[2][l][threadIdx.x]);
                float st[V];
                if (s >= 0) {
                    own.closed = 1;
                    if (p.active) load_state<V>(a.state_in, s, a.channels, p.channel, st);
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float f, k;
                    decode_gate(m[l][v], a.logit, f, k);
                    const float xv = to_float(px.e[v]);
                    const float b = outside ? 0.f : a.coupled ? xv * k : xv;
                    f = outside ? 1.f : f;
                    own.b[v] = fmaf(f, s >= 0 && p.active ? st[v] : own.b[v], b);
                    own.a[v] *= f;
                }
            }
            before = compose_warp<V, true>(own, a.lg_tx, sh_forward[stage]);
        }
        identity(own);
#pragma unroll
        for (int l = L - 1; l >= 0; --l) {
            const int e = rows.end(l);
            const bool outside = rows.outside(l);
            Pack<T, V> pd;
            if (a.v_h) pd = load_pack<T, V>(ring[stage].v[0][l][threadIdx.x]);
            float q[V];
            if (e >= 0) {
                own.closed = 1;
                if (p.active) load_state<V>(a.v_state_out, e, a.channels, p.channel, q);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float f, k;
                decode_gate(m[l][v], a.logit, f, k);
                f = outside ? 1.f : f;
                const float d = outside || !a.v_h ? 0.f : to_float(pd.e[v]);
                own.b[v] = f * (d + (e >= 0 && p.active ? q[v] : own.b[v]));
                own.a[v] *= f;
            }
        }
        const Map<V> after = compose_warp<V, false>(own, a.lg_tx, sh[stage]);
        if (TABLE && t > t0) fill_row_table(a, p0 - tile_rows, tile_rows, table(t - 1));
        __syncthreads();
        if (!APPLY) {
#pragma unroll
            for (int w = kWarps - 1; w >= 0; --w) {
                Map<V> n = warp_map<V>(sh[stage], w, p.tx);
                compose_after(n, all);
                all = n;
            }
            continue;
        }
        float h[V], q[V];
        pass_warps<V, true>(sh_forward[stage], p.tx, start, h);
        apply_map(h, before);
        pass_warps<V, false>(sh[stage], p.tx, q_carry, q);
        apply_map(q, after);
#pragma unroll
        for (int l = 0; l < L; ++l) {          // u_t: h_{t-1}, coupled: h_{t-1} - x_t
            const int s = rows.first(l);
            if (s >= 0 && p.active) load_state<V>(a.state_in, s, a.channels, p.channel, h);
            const bool outside = rows.outside(l);
            const Pack<T, V> px = load_pack<T, V>(ring[stage].v[2][l][threadIdx.x]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float f, k;
                decode_gate(m[l][v], a.logit, f, k);
                const float xv = to_float(px.e[v]);
                const float b = outside ? 0.f : a.coupled ? xv * k : xv;
                u[l][v] = a.coupled ? h[v] - xv : h[v];
                h[v] = fmaf(outside ? 1.f : f, h[v], b);
            }
        }
        const long long row = p.chain * a.chain_rows + p0 + p.row0;
        const int left = (int)min(a.chain_rows - p0 - p.row0, (long long)L);
        T* px = a.v_x ? static_cast<T*>(a.v_x) + row * a.h_stride + p.channel : nullptr;
#pragma unroll
        for (int l = L - 1; l >= 0; --l) {
            const int s = rows.first(l), e = rows.end(l);
            if (e >= 0 && p.active) load_state<V>(a.v_state_out, e, a.channels, p.channel, q);
            const bool outside = rows.outside(l) || !p.active;
            Pack<T, V> pd;
            if (a.v_h) pd = load_pack<T, V>(ring[stage].v[0][l][threadIdx.x]);
            float dx[V], dg[V], sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float f, k;
                decode_gate(m[l][v], a.logit, f, k);
                const float g = (outside || !a.v_h ? 0.f : to_float(pd.e[v])) + q[v];
                dx[v] = outside ? 0.f : a.coupled ? k * g : g;
                dg[v] = outside ? 0.f : a.logit ? g * u[l][v] * (f * k) : g * u[l][v];
                sum += dg[v];
                q[v] = outside ? q[v] : f * g;
            }
            if (px && p.active && l < left) store_floats<T, V>(px + l * a.h_stride, dx);
            if (s >= 0 && p.active && a.v_state_in) store_floats<float, V>(a.v_state_in + (long long)s * a.channels + p.channel, q);
            if (a.v_gate) {
                if (!a.shared) {
                    if (p.active && l < left) store_floats<T, V>(static_cast<T*>(a.v_gate) + (row + l) * a.gate_out_stride + p.channel, dg);
                } else {
                    for (int off = (1 << a.lg_tx) >> 1; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                    if (p.tx == 0 && l < left) {
                        const long long o = (row + l) * a.gate_out_stride + p.head;
                        if (a.parts == 1) from_float(sum, static_cast<T*>(a.v_gate)[o]);
                        else a.gate_parts[(a.reverse ? (a.rows - 1) * a.gate_heads + o : o) + (long long)p.part * a.rows * a.gate_heads] = sum;
                    }
                }
            }
        }
    }
    if (APPLY) pass_empty_sequences(a, a.v_state_out, a.v_state_in);
    else store_segment_map<V>(a, p, all);
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
        float f, k;
        decode_gate(m, logit, f, k);
        o[v] = fmaf(f, ps.e[v], coupled ? k * xv : xv);
    }
    store_floats<float, V>(state + i, o);
    store_floats<T, V>(h + i, o);
}

// ---- host ----------------------------------------------------------------------------------------------------------------

// Consecutive rows of a thread: as many as keep the backward's values of a tile in registers and two tiles of every tensor
// in shared memory with four blocks on an SM.
template <typename T> constexpr int rows_per_thread(int vec) { return vec == 4 ? (sizeof(T) == 4 ? 4 : 8) : 16; }
constexpr int kSms = 148, kBlocksPerSm = 4;

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
int shape_vec(const DsbRecurrence& s) {
    const bool shared = s.gate_heads != s.channels;
    return (shared ? s.channels / s.gate_heads : s.channels) % 4 == 0 ? 4 : 1;
}
Layout layout_of(const DsbRecurrence& s) {
    Layout l;
    l.vec = shape_vec(s);
    const bool shared = s.gate_heads != s.channels;
    l.heads = shared ? s.gate_heads : 1;
    l.per_head = s.channels / l.heads;
    const int wide = (l.per_head + l.vec - 1) / l.vec;
    const int rows = s.dtype == DSB_DTYPE_F32 ? rows_per_thread<float>(l.vec) : rows_per_thread<__half>(l.vec);
    l.lg_tx = 0;
    while (l.lg_tx < 5 && (1 << l.lg_tx) < wide) ++l.lg_tx;
    for (;;) {
        l.parts = (wide + (1 << l.lg_tx) - 1) >> l.lg_tx;
        l.tile_rows = kWarps * (32 >> l.lg_tx) * rows;
        // A chain per sequence wastes half a tile per sequence on average; a table costs a look at every row.
        l.table = s.sequence_rows == 0 || s.sequence_rows < l.tile_rows;
        l.chains = l.table ? 1 : s.sequences;
        // Narrower channel blocks where wide ones are too few to fill the GPU, down to a 64-byte piece of a row.
        if (l.lg_tx <= 3 || l.chains * l.heads * l.parts >= kSms * kBlocksPerSm) break;
        --l.lg_tx;
    }
    l.chain_rows = l.table ? s.rows : s.sequence_rows;
    l.tiles = (l.chain_rows + l.tile_rows - 1) / l.tile_rows;
    const int64_t blocks = l.chains * l.heads * l.parts;
    l.segments = 1;
    if (blocks < kSms * kBlocksPerSm / 2 && l.tiles > 1) {
        l.segments = kSms * kBlocksPerSm / blocks;
        if (l.segments > l.tiles) l.segments = l.tiles;
    }
    l.segment_tiles = l.tiles ? (l.tiles + l.segments - 1) / l.segments : 0;
    if (l.tiles) l.segments = (l.tiles + l.segment_tiles - 1) / l.segment_tiles;   // none of them empty
    return l;
}
int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }

int64_t direction_workspace(const DsbRecurrence& s, const Layout& l, bool forward) {
    const int64_t maps = l.chains * l.segments;
    int64_t bytes = 0;
    if (l.segments > 1) bytes += 2 * up16(maps * s.channels * 4) + up16(maps * 4);
    if (!forward && s.gate_heads != s.channels && l.parts > 1) bytes += up16((int64_t)l.parts * s.rows * s.gate_heads * 4);
    return bytes;
}

bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

struct Cut { Layout layout; Args args; int64_t blocks; };

int make_cut(const DsbRecurrence& s, bool forward, void* workspace, int64_t workspace_bytes, float* checkpoints, Cut* out) {
    Cut& c = *out;
    c.layout = layout_of(s);
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
    a.tiles = l.tiles; a.segments = l.segments; a.segment_tiles = l.segment_tiles;
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
    if (l.segments > 1) {
        const int64_t maps = l.chains * l.segments, bytes = up16(maps * s.channels * 4);
        a.map_a = reinterpret_cast<float*>(w); w += bytes;
        a.map_b = reinterpret_cast<float*>(w); w += bytes;
        a.map_closed = reinterpret_cast<int*>(w); w += up16(maps * 4);
    }
    if (!forward && a.shared && l.parts > 1) a.gate_parts = reinterpret_cast<float*>(w);
    c.blocks = l.chains * l.segments * l.heads * l.parts;
    DSB_REQUIRE(c.blocks <= kMaxRows, "recurrence: too many blocks for one launch");
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

template <typename Kernel>
int launch_walk(Kernel kernel, unsigned grid, size_t smem, const Args& a, cudaStream_t s) {
    if (smem > 32 * 1024)   // beside the static part
        DSB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<grid, kThreads, smem, s>>>(a);
    DSB_LAUNCH_CHECK();
    return DSB_OK;
}

template <typename T, int V, bool FORWARD>
int run_walks(const Cut& c, cudaStream_t s) {
    const Args& a = c.args;
    const bool table = c.layout.table;
    constexpr int L = rows_per_thread<T>(V);
    const size_t smem = kStages * sizeof(Stage<T, V, L, FORWARD ? 2 : 3>) + (table ? kTables * 2 * sizeof(int) * c.layout.tile_rows : 0);
    const unsigned grid = (unsigned)c.blocks;
    auto launch = [&](auto apply) {
        constexpr bool APPLY = decltype(apply)::value;
        if (FORWARD)
            return table ? launch_walk(recurrence_forward_kernel<T, V, L, true, APPLY>, grid, smem, a, s)
                         : launch_walk(recurrence_forward_kernel<T, V, L, false, APPLY>, grid, smem, a, s);
        return table ? launch_walk(recurrence_backward_kernel<T, V, L, true, APPLY>, grid, smem, a, s)
                     : launch_walk(recurrence_backward_kernel<T, V, L, false, APPLY>, grid, smem, a, s);
    };
    if (a.segments > 1) {
        const int rc = launch(std::false_type{});
        if (rc != DSB_OK) return rc;
    }
    return launch(std::true_type{});
}

template <bool FORWARD>
int run_direction(const DsbRecurrence& shape, const Cut& c, cudaStream_t s) {
    int rc = DSB_OK;
    with_dtype(shape.dtype, [&](auto tag) {
        typedef decltype(tag) T;
        rc = c.layout.vec == 4 ? run_walks<T, 4, FORWARD>(c, s) : run_walks<T, 1, FORWARD>(c, s);
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
    const Layout l = layout_of(s);
    const int64_t f = direction_workspace(s, l, true), b = direction_workspace(s, l, false);
    return f > b ? f : b;
}

int64_t recurrence_checkpoint_bytes(const DsbRecurrence& s) {
    if (check_shape(s, false) != DSB_OK) return 0;
    const Layout l = layout_of(s);
    return l.chains * l.tiles * s.channels * 4;
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
