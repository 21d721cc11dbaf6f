// The walk of the gated recurrence (recurrence.cu has its formulas and entry points), forward and backward.
//
// A stretch of rows maps the state before it to the state after it as h -> a h + b, and two stretches compose as
// (a2 a1, a2 b1 + b2); a stretch in which a sequence begins maps every h to b ("closed": its a is never looked at, so
// that an infinity of the sequence before cannot meet a zero).
//
// A block walks along one stretch of rows and a block of channels, tile by tile, and carries the state in registers: it
// reads everything once and writes everything once.  Inside a tile a thread runs L consecutive rows of V channels, and the
// threads' maps meet in shared memory, where one thread per channel passes the state through them (two barriers a tile).
// The next tile's rows are on their way into shared memory meanwhile; each thread copies what it will read itself, so their
// arrival needs no barrier.  Where sequences and channels alone make too few blocks for the GPU, a sequence is cut into
// segments: a first launch leaves every segment's map, and each block of the second starts from the composition of those
// before it.  That reads the inputs twice, the second time from L2 where the call is small enough to need it; with packed
// sequences only what lies behind a segment's last border is read twice.
//
// The backward walks from the last row to the first on q.  It needs h_{t-1}, and recomputes it in 32 bits from states that the
// forward leaves at every thread's first row (a 32-bit value per L rows and channel): the h that was written out is
// rounded to the storage type and need not be kept, and no second composition is needed.
//
// Every order of composition is fixed by the shape alone, so results do not depend on timing; no block waits for another.
//
// Measured on 8 x 4096 x 2560 bf16, per-channel logits, coupled: forward 132 us for 570 MB, backward 209 us for 906 MB
// (checkpoints included), 4.3 TB/s or 0.66 of the copy rate each.  What bounds it: instruction issue and the waits between a
// tile's phases; DRAM is 45% busy, a scheduler issues in 47% of the cycles, 24 (39) instructions an element.  What led there,
// forward + backward of that case:
//   three launches (maps, a thread per channel over all chunks, apply), everything read twice           1810 us
//   walking with the state in registers                                                                 1177
//   code of its own for tiles without a border ("plain"), gate forms compiled in, states per row group   650
//   gates kept as exp(-g): f and 1 - f from it in three instructions, without branches                   477
//   two channels an instruction, registers not spilled (L chosen for 128 registers; every large spill cost
//   more than the occupancy it bought; 8 to 12 bytes a thread remain in six 16-bit backward kernels)     327
//   blocks of 256 threads with as many threads a row as make two blocks an SM, maps through shared
//   memory: the same here, but 0.9 to 0.75 of the time with padded, packed and narrow sequences          340
// Tried and slower: three or four stages of prefetch (fewer blocks), 128 threads (row pieces below two sectors), every thread
// passing through all of a tile's maps (one barrier, 10 instructions an element more).  Without the pass through the maps
// the forward would take 114 us.
#pragma once
#include <atomic>
#include <type_traits>

#include "vector_io.cuh"

namespace dsb {

struct RecurrenceArgs {
    const void *x, *gate, *v_h;
    void *h, *v_x, *v_gate;
    const float *state_in, *v_state_out;
    float *state_out, *v_state_in;
    float* checkpoints;    // [chains][tiles][groups of L rows][channels]: the state before each group
    float *map_a, *map_b;  // [chains][segments][channels]
    int* map_closed;       // [chains][segments]
    float* gate_parts;     // [parts][rows][heads], when a head spans several channel blocks
    const int *offsets, *lengths;
    int* device_status;
    int rows, chain_rows, chains;
    // In bytes; negative when the scan runs from the last row to the first.
    long long x_stride, gate_stride, v_h_stride;   // from row to row
    long long h_stride, gate_out_stride;           // contiguous results of channels / heads
    long long x_step, gate_step, v_h_step, h_step, gate_out_step;   // from tile to tile
    int tiles, segments, segment_tiles;
    int sequences, sequence_rows, channels, gate_heads, per_head;
    int head_blocks, block_heads, head_threads;    // of a row; heads of a block; threads of a head (all tx, or a power of two)
    int parts;             // blocks that share a head
    int tx, groups;        // threads side by side on one row, groups of L rows in a tile
    int shuffle, entries;  // whether a warp composes its maps by itself, and how many maps a tile leaves in shared memory
    int reverse, table;    // table: one chain over all rows, with sequence borders anywhere; else one chain per sequence
    int logit, coupled, shared;
};
struct RecurrenceLaunch {
    RecurrenceArgs args;
    int vec, tile_rows;
    unsigned blocks;
};
template <typename T> int run_recurrence_forward(const RecurrenceLaunch& c, cudaStream_t s);
template <typename T> int run_recurrence_backward(const RecurrenceLaunch& c, cudaStream_t s);

constexpr int kWalkThreads = 256;
constexpr int kWalkWarps = kWalkThreads / 32;
constexpr int kMaxEntries = 32;

// Consecutive rows of a thread: as many as keep a tile's values in the 128 registers that two blocks on an SM leave a thread
// (a row more spills: 8 x 4096 x 2560 bf16 backward 209 -> 273 us; a row less costs 4% by more tiles), and two tiles of every
// tensor in shared memory.
template <typename T> __host__ __device__ constexpr int walk_rows(int vec) { return vec == 4 ? (sizeof(T) == 4 ? 3 : 5) : vec == 3 ? 5 : vec == 2 ? (sizeof(T) == 4 ? 6 : 8) : 12; }

// ---- V channels at a time -------------------------------------------------------------------------------------------
// Two channels an instruction where the hardware has one; `a` may be a single value for all channels.
__device__ __forceinline__ u64 pair_of(float lo, float hi) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split_pair(u64 r, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(r)); }
template <int V, int A>
__device__ __forceinline__ void mul_add(float (&r)[V], const float (&a)[A], const float (&b)[V], const float (&c)[V]) {
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
            u64 o;
            asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(o) : "l"(pair_of(a[v % A], a[(v + 1) % A])), "l"(pair_of(b[v], b[v + 1])), "l"(pair_of(c[v], c[v + 1])));
            split_pair(o, r[v], r[v + 1]);
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = fmaf(a[v % A], b[v], c[v]);
    }
}
template <int V, int A>
__device__ __forceinline__ void mul(float (&r)[V], const float (&a)[A], const float (&b)[V]) {
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
            u64 o;
            asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(o) : "l"(pair_of(a[v % A], a[(v + 1) % A])), "l"(pair_of(b[v], b[v + 1])));
            split_pair(o, r[v], r[v + 1]);
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = a[v % A] * b[v];
    }
}
template <int V, int A>
__device__ __forceinline__ void add(float (&r)[V], const float (&a)[A], const float (&b)[V]) {
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
            u64 o;
            asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(o) : "l"(pair_of(a[v % A], a[(v + 1) % A])), "l"(pair_of(b[v], b[v + 1])));
            split_pair(o, r[v], r[v + 1]);
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = a[v % A] + b[v];
    }
}

// ---- gates ---------------------------------------------------------------------------------------------------------
// A gate is kept as one register: a decay as itself, a logit g as e = exp(-g), from which f = 1 / (1 + e) and 1 - f = e f
// follow with full relative precision however close to 0 or 1 they are.  e is kept below 2^126, where 1 / (1 + e) is still a
// normal number (1.2e-38); a NaN stays one.
// Errors relative to f and to 1 - f, with u = 2^-24: 2^x by the hardware 4 u, the quotient 2 u, 1 + e and the product u each, and up
// to 1.22 |g| u by the argument g log2 e (its rounding u, the constant's own 0.22 u).  16-bit gates are left with that: at most
// 2^-17, where half a step of their type is 2^-11 or 2^-8.  32-bit gates get it back to first order from the product's and the
// constant's rests, four instructions and one rounding more: 9 u in all for |g| <= 87; beyond, e keeps its value at 87.
template <typename T, bool LOGIT, int A>
__device__ __forceinline__ void gate_registers(const Pack<T, A>& gate, float (&e)[A]) {
    float g[A];
#pragma unroll
    for (int v = 0; v < A; ++v) g[v] = to_float(gate.e[v]);
    constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147181f;
    if constexpr (!LOGIT) {
#pragma unroll
        for (int v = 0; v < A; ++v) e[v] = g[v];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int v = 0; v < A; ++v) {
            float y;
            asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, 0f42AE0000;\n\tmax.NaN.f32 %0, t, 0fC2AE0000;\n\t}" : "=f"(y) : "f"(-g[v]));   // +-87
            const float hi = y * kLog2e, lo = fmaf(y, kLog2eRest, fmaf(y, kLog2e, -hi));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[v]) : "f"(hi));
            e[v] = fmaf(e[v], lo * kLn2, e[v]);
        }
    } else {
        const float scale[1] = {-kLog2e};
        float y[A];
        mul(y, scale, g);
#pragma unroll
        for (int v = 0; v < A; ++v) {
            float t;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(y[v]));
            asm("min.NaN.f32 %0, %1, 0f7E800000;" : "=f"(e[v]) : "f"(t));
        }
    }
}
// f and k = 1 - f.  volatile: worked out again where they are used again, rather than kept in a register per element (the
// backward's values of a tile then fit the registers of more blocks on an SM).
template <bool LOGIT, int A>
__device__ __forceinline__ void gate_f(const float (&e)[A], float (&f)[A]) {
    if constexpr (!LOGIT) {
#pragma unroll
        for (int v = 0; v < A; ++v) f[v] = e[v];
    } else {
        const float one[1] = {1.f};
        float d[A];
        add(d, one, e);
#pragma unroll
        for (int v = 0; v < A; ++v) asm volatile("rcp.approx.ftz.f32 %0, %1;" : "=f"(f[v]) : "f"(d[v]));
    }
}
template <bool LOGIT, int A>
__device__ __forceinline__ void gate_k(const float (&e)[A], const float (&f)[A], float (&k)[A]) {
    if constexpr (LOGIT) {
        mul(k, e, f);
    } else {
#pragma unroll
        for (int v = 0; v < A; ++v) k[v] = 1.f - f[v];
    }
}

// ---- rows that begin and end sequences ------------------------------------------------------------------------------
// In the order of the scan: position p is row p, or rows - 1 - p when the scan runs backwards; sequence k of the scan is
// the tensor's sequence k, or sequences - 1 - k.
constexpr int kTables = 3;              // border tables: one is read, one is made, and the slowest warp may still read the one before
// Tiles in shared memory: one is worked on, one is on its way.  Flat tiles, whose rows other threads have copied and other
// threads write back, need the one before as well.
__host__ __device__ constexpr int walk_stages(int vec) { return vec == 3 ? 3 : 2; }

__device__ __forceinline__ int sequence_id(const RecurrenceArgs& a, int k) { return a.reverse ? a.sequences - 1 - k : k; }
// Where the scan's packed sequence k begins (k = sequences: where the last one ends).
__device__ __forceinline__ int packed_start(const RecurrenceArgs& a, int k) {
    const int o = a.reverse ? a.rows - min(max(a.offsets[a.sequences - k], 0), a.rows) : a.offsets[k];
    return min(max(o, 0), a.rows);   // offsets out of range are reported (pass_empty_sequences); here they must not overflow
}
// How many of packed_start(shift .. shift + sequences - 1) are <= p; called by one whole warp.
__device__ __forceinline__ int starts_up_to(const RecurrenceArgs& a, int shift, int p) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = a.sequences;
    while (len > 0) {
        const int step = (len + 31) / 32;
        const int at = min(lane, len) * step;     // 32 steps may pass 2^31
        const bool below = at >= 0 && at < len && packed_start(a, shift + lo + at) <= p;
        const int below_count = __popc(__ballot_sync(0xffffffffu, below));
        if (below_count == 0) break;
        const int skip = (below_count - 1) * step + 1;
        len = min(step - 1, len - skip);
        lo += skip;
    }
    return lo;
}

// The tiles of a segment that its map depends on: those since (FORWARD; else: until) the last sequence to begin there (the first
// to end).  Called by the whole block; narrows [t0, t1).
template <bool FORWARD>
__device__ __forceinline__ void narrow_to_map(const RecurrenceArgs& a, int tile_rows, int& t0, int& t1) {
    if (!a.table) return;
    const int last = min(t1 * tile_rows, a.rows) - 1, first = t0 * tile_rows;
    int at;
    if (a.sequence_rows > 0) {
        at = FORWARD ? last / a.sequence_rows * a.sequence_rows : first / a.sequence_rows * a.sequence_rows + (a.sequence_rows - 1);
    } else {
        __shared__ int s_found;
        if (threadIdx.x < 32) {
            int p;
            if (FORWARD) {
                const int n = starts_up_to(a, 0, last);
                p = n > 0 ? packed_start(a, n - 1) : 0;
            } else {
                const int n = starts_up_to(a, 1, first);
                p = n < a.sequences ? packed_start(a, n + 1) - 1 : a.rows;
            }
            if (threadIdx.x == 0) s_found = p;
        }
        __syncthreads();
        at = s_found;
    }
    if (FORWARD) t0 = min(max(t0, at / tile_rows), t1 - 1);
    else t1 = max(min(t1, at / tile_rows + 1), t0 + 1);
}

enum TileKind { kPlain, kBorders, kEmpty };   // no border and every row in a sequence; anything; no row in a sequence

// The borders of one tile: per group of L rows three bit masks (rows that belong to a sequence, that begin one, that end one),
// and per row with a border the sequence's id.
struct BorderTable {
    unsigned *inside, *first, *end;
    int *first_id, *end_id;
    __device__ __forceinline__ BorderTable(int* at, int groups, int tile_rows) {
        inside = reinterpret_cast<unsigned*>(at);
        first = inside + groups;
        end = first + groups;
        first_id = reinterpret_cast<int*>(end + groups);
        end_id = first_id + tile_rows;
    }
};
__host__ __device__ constexpr int table_ints(int groups, int rows_per_group) { return groups * (3 + 2 * rows_per_group); }

// Follows a walk from tile to tile (FORWARD: upwards): what kind of tile comes, and the tables of tiles with borders.  Every
// member but `window` is the same in all threads of the block.
template <bool FORWARD, int L>
struct Borders {
    int lo, hi;            // the sequence last met holds positions [lo, hi)
    int sequence;          // chain per sequence: its id.  Packed: where to look on, as a sequence of the scan
    int* tables;
    int groups, tile_rows;
    // Packed: where the sequences around the cursor begin, one per thread, loaded well before they are looked at.  FORWARD:
    // thread i has that of sequence + i; else of sequence + 1 - i.
    int window, all_begin, all_end;
    int channel, channels; // the block's channels

    // A border's states are on their way to L2 a tile before they are asked for.
    __device__ __forceinline__ void warm(const float* states, int id, int all_channels) const {
        if (!states) return;
        const char* at = reinterpret_cast<const char*>(states + (long long)id * all_channels + channel);
        for (int c = 0; c < channels * 4; c += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + c));
    }
    __device__ void begin(const RecurrenceArgs& a, int chain, int p0, int* s_tables, int lanes, int block_head, int part) {
        channel = block_head * a.per_head + part * a.tx * lanes;
        channels = min(a.tx * lanes, a.channels - channel);
        tables = s_tables;
        groups = a.groups;
        tile_rows = groups * L;
        lo = 1; hi = 0;
        if (!a.table) {
            sequence = sequence_id(a, chain);
            int len = a.sequence_rows;
            if (a.lengths) len = min(max(a.lengths[sequence], 0), a.sequence_rows);
            lo = a.reverse ? a.sequence_rows - len : 0;
            hi = lo + len;
        } else if (a.sequence_rows == 0) {
            // FORWARD: the first sequence to end after p0; else the last to begin before the tile's end
            __shared__ int s_at;
            if (threadIdx.x < 32) {
                const int n = FORWARD ? starts_up_to(a, 1, p0) : starts_up_to(a, 0, p0 + tile_rows - 1) - 1;
                if (threadIdx.x == 0) s_at = n;
            }
            __syncthreads();
            sequence = s_at;
            if (sequence >= 0 && sequence < a.sequences) {
                lo = packed_start(a, sequence);
                hi = packed_start(a, sequence + 1);
            }
            all_begin = packed_start(a, 0);
            all_end = packed_start(a, a.sequences);
            load_window(a);
        }
    }
    __device__ void load_window(const RecurrenceArgs& a) {
        const int k = FORWARD ? sequence + (int)threadIdx.x : sequence + 1 - (int)threadIdx.x;
        window = packed_start(a, min(max(k, 0), a.sequences));
    }
    __device__ __forceinline__ BorderTable table(int t) const {
        return BorderTable(tables + t % kTables * table_ints(groups, L), groups, tile_rows);
    }
    // The rows of the group at p that lie in [from, to).
    __device__ __forceinline__ static unsigned mask_of(int p, int from, int to) {
        const int b = min(max(from - p, 0), L), e = min(max(to - p, 0), L);
        return b < e ? ((1u << e) - 1u) & ~((1u << b) - 1u) : 0u;
    }

    // Tile t at p0; called by the whole block, tile after tile.  Tables are there after the next barrier.
    __device__ int prepare(const RecurrenceArgs& a, int t, int p0) {
        const int p1 = p0 + tile_rows;
        if (p0 > lo && p1 < hi) return kPlain;
        if (!a.table && (p1 <= lo || p0 >= hi)) return kEmpty;
        const BorderTable b = table(t);
        const int tid = threadIdx.x, p = p0 + tid * L;      // one thread per group
        if (!a.table) {
            if (tid < groups) {
                const int last = lo < hi ? hi - 1 : -1;     // a sequence of no rows ends nowhere
                b.inside[tid] = mask_of(p, lo, hi);
                b.first[tid] = lo < hi ? mask_of(p, lo, lo + 1) : 0u;
                b.end[tid] = mask_of(p, last, last + 1);
                if (lo >= p && lo < p + L) b.first_id[lo - p0] = sequence;
                if (last >= p && last < p + L) b.end_id[last - p0] = sequence;
            }
            return kBorders;
        }
        if (a.sequence_rows > 0) {
            if (tid < groups) {
                unsigned inside = 0, first = 0, end = 0;
                for (int l = 0; l < L && p + l < a.rows; ++l) {
                    const int turn = (p + l) / a.sequence_rows, pos = p + l - turn * a.sequence_rows;
                    const int seq = sequence_id(a, turn);
                    const int len = a.lengths ? min(max(a.lengths[seq], 0), a.sequence_rows) : a.sequence_rows;
                    const int at = a.reverse ? a.sequence_rows - len : 0;
                    if (pos < at || pos >= at + len) continue;
                    inside |= 1u << l;
                    if (pos == at) { first |= 1u << l; b.first_id[tid * L + l] = seq; }
                    if (pos == at + len - 1) { end |= 1u << l; b.end_id[tid * L + l] = seq; }
                }
                b.inside[tid] = inside;
                b.first[tid] = first;
                b.end[tid] = end;
            }
            return kBorders;
        }
        const int last = min(p1, a.rows);
        if (tid < groups) {
            b.inside[tid] = mask_of(p, all_begin, min(all_end, last));
            b.first[tid] = 0;
            b.end[tid] = 0;
        }
        __shared__ int s_window[kWalkThreads];
        int done;
        do {   // offsets out of order may lead this astray, but every access stays where it belongs
            s_window[tid] = window;
            __syncthreads();
            const int k = FORWARD ? sequence + tid : sequence - tid;
            bool through = false;
            if (tid < kWalkThreads - 1 && k >= 0 && k < a.sequences) {
                const int o0 = FORWARD ? window : s_window[tid + 1], o1 = FORWARD ? s_window[tid + 1] : window;
                if (o0 < o1) {
                    const int id = sequence_id(a, k);
                    if (o0 >= p0 && o0 < last) {
                        b.first_id[o0 - p0] = id;
                        warm(a.state_in, id, a.channels);
                        atomicOr(&b.first[(o0 - p0) / L], 1u << ((o0 - p0) % L));
                    }
                    if (o1 > p0 && o1 <= last) {
                        b.end_id[o1 - 1 - p0] = id;
                        if (!FORWARD) warm(a.v_state_out, id, a.channels);
                        atomicOr(&b.end[(o1 - 1 - p0) / L], 1u << ((o1 - 1 - p0) % L));
                    }
                }
                through = FORWARD ? o1 <= p1 : o0 >= p0;
            }
            done = __syncthreads_count(through);
            sequence += FORWARD ? done : -done;
            const bool any = done < kWalkThreads - 1 && sequence >= 0 && sequence < a.sequences;
            const int w0 = any ? s_window[done] : 0, w1 = any ? s_window[done + 1] : 0;
            lo = any ? (FORWARD ? w0 : w1) : 1;
            hi = any ? (FORWARD ? w1 : w0) : 0;
            load_window(a);
            if (done == kWalkThreads - 1) __syncthreads();   // the window is about to be overwritten
        } while (done == kWalkThreads - 1);
        return kBorders;
    }
};

// Sequences without rows hand their state on; offsets and lengths out of order or range are reported.  Neighbours in the list go
// to different blocks, and a warp copies what its lanes have found.
__device__ __forceinline__ void pass_empty_sequences(const RecurrenceArgs& a, const float* in, float* out) {
    if (!a.offsets && !a.lengths) return;
    const int lane = threadIdx.x & 31;
    const long long step = (long long)gridDim.x * kWalkThreads;
    for (long long s0 = blockIdx.x + (long long)(threadIdx.x & ~31) * gridDim.x; s0 < a.sequences; s0 += step) {
        const long long s = s0 + (long long)lane * gridDim.x;
        bool empty = false, bad = false;
        if (s < a.sequences) {
            if (a.offsets) {
                const long long o0 = a.offsets[s], o1 = a.offsets[s + 1];
                empty = o1 <= o0;
                bad = o1 < o0 || o0 < 0 || o1 > a.rows;
            } else {
                const int len = a.lengths[s];
                empty = len <= 0;
                bad = len < 0 || len > a.sequence_rows;
            }
        }
        if (bad) atomicMin(a.device_status, DSB_ERR_INVALID_ARGUMENT);
        unsigned left = __ballot_sync(0xffffffffu, (empty || bad) && out);
        while (left) {
            const long long at = (s0 + (long long)(__ffs(left) - 1) * gridDim.x) * a.channels;
            left &= left - 1;
#pragma unroll 8
            for (int c = lane; c < a.channels; c += 32) out[at + c] = in ? __ldg(in + at + c) : 0.f;
        }
    }
}

// ---- maps and their composition ----------------------------------------------------------------------------------------
// A is V, or 1 where all channels of a thread share the gate.
template <int V, int A>
struct Map {
    float a[A], b[V];
    int closed;
};
template <int V, int A>
__device__ __forceinline__ void identity(Map<V, A>& m) {
#pragma unroll
    for (int v = 0; v < A; ++v) m.a[v] = 1.f;
#pragma unroll
    for (int v = 0; v < V; ++v) m.b[v] = 0.f;
    m.closed = 0;
}
// m <- m after e (e comes first along the scan).  PLAIN: neither is closed.
template <bool PLAIN, int V, int A>
__device__ __forceinline__ void compose_after(Map<V, A>& m, const Map<V, A>& e) {
    const bool open = PLAIN || !m.closed;
    float b[V];
    mul_add(b, m.a, e.b, m.b);
#pragma unroll
    for (int v = 0; v < V; ++v) m.b[v] = open ? b[v] : m.b[v];
    mul(m.a, e.a, m.a);
    if (!PLAIN) m.closed |= e.closed;
}
template <bool PLAIN, int V, int A>
__device__ __forceinline__ void apply_map(float (&h)[V], const Map<V, A>& m) {
    float n[V];
    mul_add(n, m.a, h, m.b);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = PLAIN || !m.closed ? n[v] : m.b[v];
}

// The maps of one tile in shared memory, in the order of its rows: one per group of rows, or one per warp.
template <int V, int A>
struct alignas(16) TileMaps {     // read and written V (A) floats at a time
    float b[kWalkThreads * V];
    float a[kWalkThreads * A];
    int closed[kMaxEntries];
};
template <bool PLAIN, int V, int A>
__device__ __forceinline__ void put_map(TileMaps<V, A>& sh, int entry, int tx_count, int tx, const Map<V, A>& m) {
    const int at = entry * tx_count + tx;
    store_floats<float, A>(&sh.a[at * A], m.a);
    store_floats<float, V>(&sh.b[at * V], m.b);
    if (!PLAIN && tx == 0) sh.closed[entry] = m.closed;
}
template <bool PLAIN, int V, int A>
__device__ __forceinline__ Map<V, A> get_map(const TileMaps<V, A>& sh, int entry, int tx_count, int tx) {
    Map<V, A> m;
    const int at = entry * tx_count + tx;
    const Pack<float, A> pa = load_pack<float, A>(&sh.a[at * A]);
    const Pack<float, V> pb = load_pack<float, V>(&sh.b[at * V]);
#pragma unroll
    for (int v = 0; v < A; ++v) m.a[v] = pa.e[v];
#pragma unroll
    for (int v = 0; v < V; ++v) m.b[v] = pb.e[v];
    m.closed = PLAIN ? 0 : sh.closed[entry];
    return m;
}

// ---- a block's place -----------------------------------------------------------------------------------------------------
// Where many threads share a row, every group of rows leaves its map in shared memory (any number of threads a row, so that
// the blocks can be made as many as the SMs hold).  Where few do (1, 2, 4 or 8), groups are many: a warp composes its own.
struct Place {
    int chain, segment, part, tx;
    int block_head, head, channel;   // the block's first head; this thread's, and its first channel
    int row0, group;       // this thread's first row inside a tile, and which of the tile's groups of rows that is
    int entry;             // whose map in shared memory includes this thread's rows
    bool there, active;    // there: one of the tile's groups; active: and not beyond the head's last channel or the last head
    bool leads;            // the first thread of a head
    int read_channel;      // what to read all the same where a thread has no channel
};
template <int V, int L, bool SHARED>
__device__ __forceinline__ Place place_of(const RecurrenceArgs& a) {
    Place p;
    const int blocks = a.head_blocks * a.parts;
    const int rest = (int)(blockIdx.x / (unsigned)blocks);
    const int block = (int)(blockIdx.x - (unsigned)rest * blocks);
    p.segment = rest / a.chains;
    p.chain = rest - p.segment * a.chains;
    const int head_block = block / a.parts;
    p.part = block - head_block * a.parts;
    p.block_head = head_block * a.block_heads;
    const int tid = threadIdx.x;
    p.group = tid / a.tx;
    p.tx = tid - p.group * a.tx;
    p.there = p.group < a.groups;
    if (!p.there) p.group = 0;
    p.entry = a.shuffle ? tid >> 5 : p.group;
    p.row0 = p.group * L;
    // Without shared gates the same arithmetic with one head: any shorter form of it made the coupled backward of four 16-bit
    // channels a thread spill 130 bytes (8 x 4096 x 2560, a training pass: 348 -> 392 us).
    if (SHARED) {
        const int within = p.tx / a.head_threads, lane = p.tx - within * a.head_threads;
        const int c = (p.part * a.head_threads + lane) * V;
        p.head = p.block_head + within;
        p.channel = p.head * a.per_head + c;
        p.active = p.there && c < a.per_head && p.channel < a.channels;
        p.leads = lane == 0 && p.active;
        p.read_channel = p.active ? p.channel : p.block_head * a.per_head;
        if (p.channel >= a.channels) p.head = p.block_head;   // its gates are read and not used
    } else {
        const int c = (p.part * a.tx + p.tx) * V;
        p.head = p.block_head;
        p.active = p.there && c < a.per_head;
        p.leads = false;
        p.channel = p.head * a.per_head + c;
        p.read_channel = p.active ? p.channel : p.head * a.per_head;
    }
    return p;
}

// From every thread's own map: the tile's maps in shared memory (to be read after the next barrier), and the map of the rows
// of its entry before its own.  FORWARD: rows run with the lanes; else against them.
template <bool FORWARD, bool PLAIN, int V, int A>
__device__ __forceinline__ Map<V, A> publish_map(const RecurrenceArgs& a, const Place& p, const Map<V, A>& own, TileMaps<V, A>& sh) {
    Map<V, A> before;
    identity(before);
    if (!a.shuffle) {
        if (p.there) put_map<PLAIN>(sh, p.entry, a.tx, p.tx, own);
        return before;
    }
    const int lane = threadIdx.x & 31, tx = a.tx;
    Map<V, A> run = own;
    auto from = [&](auto value, int off) {
        return FORWARD ? __shfl_up_sync(0xffffffffu, value, off) : __shfl_down_sync(0xffffffffu, value, off);
    };
#pragma unroll 1
    for (int off = tx; off < 32; off <<= 1) {
        Map<V, A> e;
#pragma unroll
        for (int v = 0; v < A; ++v) e.a[v] = from(run.a[v], off);
#pragma unroll
        for (int v = 0; v < V; ++v) e.b[v] = from(run.b[v], off);
        e.closed = PLAIN ? 0 : from(run.closed, off);
        if (FORWARD ? lane >= off : lane + off < 32) compose_after<PLAIN>(run, e);
    }
    if (FORWARD ? lane >= 32 - tx : lane < tx) put_map<PLAIN>(sh, p.entry, tx, p.tx, run);
#pragma unroll
    for (int v = 0; v < A; ++v) before.a[v] = from(run.a[v], tx);
#pragma unroll
    for (int v = 0; v < V; ++v) before.b[v] = from(run.b[v], tx);
    if (!PLAIN) before.closed = from(run.closed, tx);
    if (FORWARD ? lane < tx : lane >= 32 - tx) identity(before);
    return before;
}
// Once a tile's maps are published: the first `tx` threads carry the state through them in their order and leave every entry's
// starting state in the place of its b.  Nobody else needs the state between tiles.  Two barriers a tile, but the
// composition costs the block one thread's work per channel instead of every thread's.  The second barrier is the caller's.
template <bool FORWARD, bool PLAIN, int V, int A>
__device__ __forceinline__ void pass_entries(const RecurrenceArgs& a, const Place& p, TileMaps<V, A>& sh, float (&carry)[V]) {
    if (threadIdx.x < a.tx) {
#pragma unroll 4
        for (int i = 0; i < a.entries; ++i) {
            const int w = FORWARD ? i : a.entries - 1 - i;
            const Map<V, A> m = get_map<PLAIN>(sh, w, a.tx, p.tx);
            store_floats<float, V>(&sh.b[(w * a.tx + p.tx) * V], carry);
            apply_map<PLAIN>(carry, m);
        }
    }
}
template <int V, int A>
__device__ __forceinline__ void entry_state(const RecurrenceArgs& a, const Place& p, const TileMaps<V, A>& sh, float (&h)[V]) {
    const Pack<float, V> q = load_pack<float, V>(&sh.b[(p.entry * a.tx + p.tx) * V]);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = q.e[v];
}
// all: the map of the tiles before (along the scan) -> that of this one as well.
template <bool FORWARD, bool PLAIN, int V, int A>
__device__ __forceinline__ void pass_entries(const RecurrenceArgs& a, const Place& p, const TileMaps<V, A>& sh, Map<V, A>& all) {
    if (threadIdx.x >= a.tx) return;
    const int closed = all.closed;
#pragma unroll 2
    for (int i = 0; i < a.entries; ++i) {
        Map<V, A> m = get_map<PLAIN>(sh, FORWARD ? i : a.entries - 1 - i, a.tx, p.tx);
        compose_after<PLAIN>(m, all);
        all = m;
    }
    if (PLAIN) all.closed = closed;
}

// The states at the borders among a thread's rows, taken one after the other (FORWARD: upwards).  The next one is asked for
// when the one before is taken, the first before the thread begins with its rows.
template <bool FORWARD, int V>
struct BorderStates {
    float next[V];
    unsigned left;
    const float* states;
    const int* ids;
    int channels, channel;
    __device__ __forceinline__ BorderStates(const float* s, unsigned mask, const int* who, int count, int at)
        : left(mask), states(s), ids(who), channels(count), channel(at) {
        ask();
    }
    __device__ __forceinline__ void ask() {
#pragma unroll
        for (int v = 0; v < V; ++v) next[v] = 0.f;
        if (left == 0) return;
        const int l = FORWARD ? __ffs(left) - 1 : 31 - __clz(left);
        left &= ~(1u << l);
        if (states) {
            const Pack<float, V> q = load_pack<float, V>(states + (long long)ids[l] * channels + channel);
#pragma unroll
            for (int v = 0; v < V; ++v) next[v] = q.e[v];
        }
    }
    __device__ __forceinline__ void take(float (&h)[V]) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = next[v];
        ask();
    }
};
// What a thread knows of its rows of one tile.
template <bool PLAIN>
struct RowBorders {
    unsigned inside, first, end;
    const int *first_id, *end_id;
    __device__ __forceinline__ RowBorders(const BorderTable& t, const Place& p) {
        inside = t.inside[p.group];
        first = t.first[p.group];
        end = t.end[p.group];
        first_id = t.first_id + p.row0;
        end_id = t.end_id + p.row0;
    }
    __device__ __forceinline__ bool is_outside(int l) const { return !(inside >> l & 1u); }
    __device__ __forceinline__ bool begins(int l) const { return first >> l & 1u; }
    __device__ __forceinline__ bool ends(int l) const { return end >> l & 1u; }
};
template <>
struct RowBorders<true> {      // a plain tile: all inside, no borders
    static constexpr unsigned first = 0, end = 0;
    const int *first_id = nullptr, *end_id = nullptr;
    __device__ __forceinline__ RowBorders(const BorderTable&, const Place&) {}
    __device__ __forceinline__ bool is_outside(int) const { return false; }
    __device__ __forceinline__ bool begins(int) const { return false; }
    __device__ __forceinline__ bool ends(int) const { return false; }
};

// ---- rows on their way through shared memory ---------------------------------------------------------------------------
template <typename T, int V>
__device__ __forceinline__ void copy_async(unsigned to, const T* from, bool there) {
    constexpr int kBytes = V * sizeof(T);
    const int bytes = there ? kBytes : 0;         // what is not copied is filled with zeros
    if (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else if (kBytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Lanes lie side by side, so that neither the copies nor the reads meet a bank twice.
template <typename T> __host__ __device__ constexpr unsigned walk_tensor_bytes(int vec) {
    return walk_rows<T>(vec) * kWalkThreads * vec * sizeof(T);
}
template <typename T, int V, int L, int TENSORS>
struct alignas(16) TileStage {
    T v[TENSORS][L][kWalkThreads][V];
};

// A thread's first element of a tile, as a byte address.
template <typename T, typename Byte>
__device__ __forceinline__ Byte* row_pointer(Byte* base, int channel, long long stride, const RecurrenceArgs& a, const Place& p, int tile,
                                             int tile_rows) {
    return base + ((long long)p.chain * a.chain_rows + (long long)tile * tile_rows + p.row0) * stride + channel * (long long)sizeof(T);
}
// The thread's rows of a tile, `left` of them within the chain (L: all, known to the whole block); the others become zeros.
// Rows that belong to no sequence but lie within the tensor are copied like the others and masked where they are used.
template <typename T, int V, int L>
__device__ __forceinline__ void fetch_rows(unsigned to, const char* from, const long long& stride, bool full, int left, const char* base) {
    constexpr unsigned kRow = kWalkThreads * V * sizeof(T);
    if (full) {
#pragma unroll
        for (int l = 0; l < L; ++l, from += stride) copy_async<T, V>(to + l * kRow, reinterpret_cast<const T*>(from), true);
    } else {
#pragma unroll 1
        for (int l = 0; l < L; ++l) copy_async<T, V>(to + l * kRow, reinterpret_cast<const T*>(l < left ? from + l * stride : base), l < left);
    }
}
// Single 16-bit elements are below what an asynchronous copy takes: loaded, all tensors' rows together, and stored.
template <typename T, int L>
struct NarrowRows {
    T v[L];
    __device__ __forceinline__ void load(const char* from, const long long& stride, int left) {
#pragma unroll
        for (int l = 0; l < L; ++l) {
            memset(&v[l], 0, sizeof(T));
            if (l < left) v[l] = *reinterpret_cast<const T*>(from + l * stride);
        }
    }
    __device__ __forceinline__ void store(unsigned char* stage) const {
#pragma unroll
        for (int l = 0; l < L; ++l) reinterpret_cast<T*>(stage)[l * kWalkThreads + threadIdx.x] = v[l];
    }
};
// A gate that channels share is read directly, as every thread of a row wants the same value.
template <typename T, int L>
__device__ __forceinline__ void fetch_shared_gates(T (&own)[L], const char* from, const long long& stride, int left) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
        memset(&own[l], 0, sizeof(T));
        if (l < left) own[l] = *reinterpret_cast<const T*>(from + l * stride);
    }
}

// The state (or q) at the segment's beginning: the maps of the segments before it, each entry a share of them, in order.
template <bool FORWARD, int V, int A>
__device__ void carry_of_segment(const RecurrenceArgs& a, const Place& p, TileMaps<V, A>& sh, float (&carry)[V]) {
    const int before = FORWARD ? p.segment : a.segments - 1 - p.segment;
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = 0.f;
    if (before == 0) return;
    const long long first_map = (long long)p.chain * a.segments;
    auto map_at = [&](int i) { return first_map + (FORWARD ? i : a.segments - 1 - i); };
    int from = 0;
    if (a.table) {         // only what follows the last segment with a border counts
        __shared__ int s_from;
        if (threadIdx.x == 0) s_from = 0;
        __syncthreads();
        for (int i = before - 1 - (int)threadIdx.x; i >= 0; i -= kWalkThreads)
            if (a.map_closed[map_at(i)]) {
                atomicMax(&s_from, i);
                break;
            }
        __syncthreads();
        from = s_from;
    }
    const int share = (before - from + a.entries - 1) / a.entries;
    const int i0 = min(from + share * p.entry, before), i1 = min(i0 + share, before);
    if (p.there && (!a.shuffle || (threadIdx.x & 31) < a.tx)) {
        Map<V, A> all;
        identity(all);
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const long long at = map_at(i);
            Map<V, A> m;
            const Pack<float, V> pa = load_pack<float, V>(a.map_a + at * a.channels + p.read_channel);
            const Pack<float, V> pb = load_pack<float, V>(a.map_b + at * a.channels + p.read_channel);
#pragma unroll
            for (int v = 0; v < A; ++v) m.a[v] = pa.e[v];
#pragma unroll
            for (int v = 0; v < V; ++v) m.b[v] = pb.e[v];
            m.closed = a.map_closed[at];
            compose_after<false>(m, all);
            all = m;
        }
        put_map<false>(sh, p.entry, a.tx, p.tx, all);
    }
    __syncthreads();
    pass_entries<true, false>(a, p, sh, carry);   // only the first threads' carry counts
    __syncthreads();
}

// Leaves the composition of a whole segment's tiles.
template <int V, int A>
__device__ __forceinline__ void store_segment_map(const RecurrenceArgs& a, const Place& p, const Map<V, A>& all) {
    if (threadIdx.x >= a.tx || !p.active) return;
    const long long at = (long long)p.chain * a.segments + p.segment;
    float wide[V];
#pragma unroll
    for (int v = 0; v < V; ++v) wide[v] = all.a[v % A];
    store_floats<float, V>(a.map_a + at * a.channels + p.channel, wide);
    store_floats<float, V>(a.map_b + at * a.channels + p.channel, all.b);
    if (p.tx == 0) a.map_closed[at] = all.closed;
}

// Flat tiles: three channels, contiguous rows, one thread per row.  Rows of 12 bytes are too narrow to be copied thread by
// thread (every access would touch 32 sectors), so the block copies a tile as the one piece of memory that it is.
struct FlatPiece {
    long long offset;      // of the piece's lowest address, in bytes from the scan's base
    int rows;
    __device__ __forceinline__ FlatPiece(const RecurrenceArgs& a, const Place& p, int p0, int tile_rows, long long stride) {
        rows = min(tile_rows, a.chain_rows - p0);
        const long long at = (long long)p.chain * a.chain_rows + p0;
        offset = (a.reverse ? at + rows - 1 : at) * stride;
    }
    // Where the scan's row r of the tile lies in the piece.
    __device__ __forceinline__ int row(const RecurrenceArgs& a, int r) const { return a.reverse ? rows - 1 - r : r; }
};
template <int L>
__device__ __forceinline__ void fetch_flat(unsigned to, const char* base, const FlatPiece& piece) {
    const float* from = reinterpret_cast<const float*>(base + piece.offset) + threadIdx.x;
    const int count = piece.rows * 3 - (int)threadIdx.x;
#pragma unroll
    for (int i = 0; i < 3 * L; ++i)
        if (i * kWalkThreads < count) copy_async<float, 1>(to + i * kWalkThreads * 4, from + i * kWalkThreads, true);
}
template <int L>
__device__ __forceinline__ void write_flat(char* base, const FlatPiece& piece, const float* from) {
    float* to = reinterpret_cast<float*>(base + piece.offset) + threadIdx.x;
    const int count = piece.rows * 3 - (int)threadIdx.x;
#pragma unroll
    for (int i = 0; i < 3 * L; ++i)
        if (i * kWalkThreads < count) to[i * kWalkThreads] = from ? from[i * kWalkThreads + threadIdx.x] : 0.f;
}

// A tile of rows that belong to no sequence.
template <typename T, int V, int L>
__device__ __forceinline__ void store_zero_rows(char* to, long long stride, int left) {
    const float zero[V] = {};
#pragma unroll 1
    for (int l = 0; l < L; ++l)
        if (l < left) store_floats<T, V>(reinterpret_cast<T*>(to + l * stride), zero);
}

template <typename T, int V, bool LOGIT, bool COUPLED, bool SHARED, bool APPLY>
__global__ void __launch_bounds__(kWalkThreads, 2)
recurrence_forward_kernel(const RecurrenceArgs a) {
    constexpr int L = walk_rows<T>(V), A = SHARED ? 1 : V, STAGES = walk_stages(V);
    constexpr bool FLAT = V == 3;
    typedef TileStage<T, V, L, SHARED ? 1 : 2> Ring;
    extern __shared__ __align__(16) unsigned char s_raw[];
    Ring* ring = reinterpret_cast<Ring*>(s_raw);
    __shared__ TileMaps<V, A> sh[2];
    const int tile_rows = a.groups * L;
    const Place p = place_of<V, L, SHARED>(a);
    int t0 = p.segment * a.segment_tiles, t1 = min(t0 + a.segment_tiles, a.tiles);
    if (!APPLY) narrow_to_map<true>(a, tile_rows, t0, t1);
    const char* x = row_pointer<T>(static_cast<const char*>(a.x), p.read_channel, a.x_stride, a, p, t0, tile_rows);
    const char* gate = row_pointer<T>(static_cast<const char*>(a.gate), SHARED ? p.head : p.read_channel, a.gate_stride, a, p, t0, tile_rows);
    const unsigned s_ring = (unsigned)__cvta_generic_to_shared(s_raw) + threadIdx.x * (FLAT ? 1 : V) * sizeof(T);
    constexpr unsigned kTensor = L * kWalkThreads * V * sizeof(T);
    const int groups = a.groups;
    const bool wanted = APPLY && a.h && p.active;
    char* to_h = row_pointer<T>(static_cast<char*>(a.h), p.channel, a.h_stride, a, p, t0, tile_rows);
    const bool keep = APPLY && a.checkpoints && p.active;
    float* to_start = a.checkpoints + (((long long)p.chain * a.tiles + t0) * groups + p.group) * a.channels + p.channel;

    float carry[V];
    Map<V, A> all;
    identity(all);
    if (APPLY) carry_of_segment<true>(a, p, sh[0], carry);
    Borders<true, L> borders;
    borders.begin(a, p.chain, t0 * tile_rows, reinterpret_cast<int*>(s_raw + STAGES * sizeof(Ring)), V, p.block_head, p.part);
    T gate_now[L], gate_next[L];
    // Fetches tile t, the next of the walk, into the stage `fetched` and moves on; tiles without rows of a sequence are only
    // passed.
    int fetched = 0;
    auto fetch = [&](int t) {
        int kind = kEmpty;
        if (t < t1) {
            kind = borders.prepare(a, t, t * tile_rows);
            if (kind != kEmpty) {
                if constexpr (FLAT) {
                    const FlatPiece piece(a, p, t * tile_rows, tile_rows, a.h_stride);
                    fetch_flat<L>(s_ring + fetched * sizeof(Ring), static_cast<const char*>(a.x), piece);
                    if (!SHARED) fetch_flat<L>(s_ring + fetched * sizeof(Ring) + kTensor, static_cast<const char*>(a.gate), piece);
                } else {
                    const int rest = a.chain_rows - t * tile_rows;
                    const int left = min(rest - p.row0, L);
                    if constexpr (V * sizeof(T) == 2) {
                        NarrowRows<T, L> rx, rg;
                        rx.load(x, a.x_stride, left);
                        if (!SHARED) rg.load(gate, a.gate_stride, left);
                        unsigned char* to = s_raw + fetched * sizeof(Ring);
                        rx.store(to);
                        if (!SHARED) rg.store(to + kTensor);
                    } else {
                        const unsigned to = s_ring + fetched * sizeof(Ring);
                        fetch_rows<T, V, L>(to, x, a.x_stride, rest >= tile_rows, left, static_cast<const char*>(a.x));
                        if (!SHARED) fetch_rows<T, V, L>(to + kTensor, gate, a.gate_stride, rest >= tile_rows, left, static_cast<const char*>(a.gate));
                    }
                }
            }
            x += a.x_step;
            if (!SHARED) gate += a.gate_step;
        }
        fetched = fetched + 1 == STAGES ? 0 : fetched + 1;
        copies_issued();
        return kind;
    };
    auto fetch_gates = [&](int t) {
        fetch_shared_gates<T, L>(gate_next, gate, a.gate_stride, t < t1 ? min(a.chain_rows - t * tile_rows - p.row0, L) : 0);
        gate += a.gate_step;
    };
    int kind = fetch(t0), kind_next = kEmpty, written = -1;   // written: a flat tile whose h waits in shared memory
    if (SHARED) fetch_gates(t0);
    if (FLAT) copies_landed<0>();
    __syncthreads();
    int stage = 0, stage_written = 0;
    auto write_back = [&] {
        if (written >= 0) write_flat<L>(static_cast<char*>(a.h), FlatPiece(a, p, written * tile_rows, tile_rows, a.h_stride), reinterpret_cast<const float*>(&ring[stage_written]));
        written = -1;
    };
    for (int t = t0; t < t1; ++t, kind = kind_next, stage = stage + 1 == STAGES ? 0 : stage + 1, to_h += a.h_step,
             to_start += (long long)groups * a.channels) {
        const int p0 = t * tile_rows;
        if (SHARED) {
#pragma unroll
            for (int l = 0; l < L; ++l) gate_now[l] = gate_next[l];
            fetch_gates(t + 1);
        }
        kind_next = fetch(t + 1);
        if (!FLAT) copies_landed<1>();
        const int left = min(a.chain_rows - p0 - p.row0, L);
        if (kind == kEmpty) {
            if constexpr (FLAT) {
                if (APPLY && a.h) write_flat<L>(static_cast<char*>(a.h), FlatPiece(a, p, p0, tile_rows, a.h_stride), nullptr);
                copies_landed<0>();
            } else if (wanted) {
                store_zero_rows<T, V, L>(to_h, a.h_stride, left);
            }
            __syncthreads();
            if (FLAT) {
                write_back();
                __syncthreads();    // before its stage is filled again
            }
            continue;
        }
        const FlatPiece piece(a, p, p0, tile_rows, a.h_stride);
        // This thread's row l of tensor k; rows of a flat tile past the chain's end give any row's values, masked like others.
        auto row_at = [&](int k, int l) {
            if constexpr (FLAT) return &ring[stage].v[0][0][0][0] + k * (L * kWalkThreads * V) + max(piece.row(a, p.row0 + l), 0) * V;
            else return &ring[stage].v[k][l][threadIdx.x][0];
        };
        auto tile = [&](auto plain) {
            constexpr bool PLAIN = decltype(plain)::value;
            const RowBorders<PLAIN> rows(borders.table(t), p);
            float f[L][A], b[L][V];
            Map<V, A> own;
            identity(own);
            BorderStates<true, V> begins(p.active ? a.state_in : nullptr, rows.first, rows.first_id, a.channels, p.channel);
            BorderStates<true, V> again = begins;       // for the second time through the rows, the first state already there
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const bool outside = rows.is_outside(l);
                const Pack<T, V> px = load_pack<T, V>(row_at(0, l));
                Pack<T, A> pg;
                if (SHARED) pg.e[0] = gate_now[l];
                else pg = load_pack<T, A>(row_at(SHARED ? 0 : 1, l));
                if (rows.begins(l)) {  // the state before this row is the sequence's own, whatever came before
                    begins.take(own.b);
                    own.closed = 1;
                }
                float e[A], k[A], xv[V];
                gate_registers<T, LOGIT>(pg, e);
                gate_f<LOGIT>(e, f[l]);
#pragma unroll
                for (int v = 0; v < V; ++v) xv[v] = to_float(px.e[v]);
                if (COUPLED) {
                    gate_k<LOGIT>(e, f[l], k);
                    mul(b[l], k, xv);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) b[l][v] = xv[v];
                }
                if (outside) {
#pragma unroll
                    for (int v = 0; v < A; ++v) f[l][v] = 1.f;
#pragma unroll
                    for (int v = 0; v < V; ++v) b[l][v] = 0.f;
                }
                mul(own.a, f[l], own.a);
                mul_add(own.b, f[l], own.b, b[l]);
            }
            const Map<V, A> before = publish_map<true, PLAIN>(a, p, own, sh[t & 1]);
            if (FLAT) copies_landed<0>();
            __syncthreads();
            if (FLAT) write_back();
            if (!APPLY) {
                pass_entries<true, PLAIN>(a, p, sh[t & 1], all);
                return;
            }
            float h[V];
            pass_entries<true, PLAIN>(a, p, sh[t & 1], carry);
            __syncthreads();
            entry_state(a, p, sh[t & 1], h);
            if (a.shuffle) apply_map<PLAIN>(h, before);
            store_floats_if<float, V>(to_start, h, keep);
            [[maybe_unused]] char* to = to_h;
#pragma unroll
            for (int l = 0; l < L; ++l) {
                if (rows.begins(l)) again.take(h);
                float o[V];
                mul_add(h, f[l], h, b[l]);
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] = rows.is_outside(l) ? 0.f : h[v];
                if constexpr (FLAT) {
                    store_floats_if<T, V>(row_at(0, l), o, wanted && (PLAIN || l < left));
                } else {
                    store_floats_if<T, V>(reinterpret_cast<T*>(to), o, wanted && (PLAIN || l < left));
                    to += a.h_stride;
                }
                if (rows.ends(l) && p.active) store_floats<float, V>(a.state_out + (long long)rows.end_id[l] * a.channels + p.channel, h);
            }
        };
        if (kind == kPlain) tile(std::true_type{});
        else tile(std::false_type{});
        if (FLAT && APPLY && a.h) {
            written = t;
            stage_written = stage;
        }
    }
    if (FLAT) {
        __syncthreads();
        write_back();
    }
    if (APPLY) pass_empty_sequences(a, a.state_in, a.state_out);
    else store_segment_map(a, p, all);
}

template <typename T, int V, bool LOGIT, bool COUPLED, bool SHARED, bool APPLY>
__global__ void __launch_bounds__(kWalkThreads, 2)
recurrence_backward_kernel(const RecurrenceArgs a) {
    constexpr int L = walk_rows<T>(V), A = SHARED ? 1 : V, STAGES = walk_stages(V);
    constexpr bool FLAT = V == 3;
    // What lies in a stage, in this order; v_h last, as it may be missing: then one tensor of zeros stands for every stage's.
    constexpr int kXAt = 0, kGateAt = APPLY ? 1 : 0, kVhAt = kGateAt + (SHARED ? 0 : 1);
    constexpr unsigned kTensor = walk_tensor_bytes<T>(V);
    const unsigned stage_bytes = (kVhAt + (a.v_h ? 1 : 0)) * kTensor;
    extern __shared__ __align__(16) unsigned char s_raw[];
    unsigned char* s_zeros = s_raw + STAGES * stage_bytes;
    __shared__ TileMaps<V, A> sh[2];
    const int tile_rows = a.groups * L;
    const Place p = place_of<V, L, SHARED>(a);
    int t0 = p.segment * a.segment_tiles, t1 = min(t0 + a.segment_tiles, a.tiles);
    if (!APPLY) narrow_to_map<false>(a, tile_rows, t0, t1);
    const char* vh = row_pointer<T>(static_cast<const char*>(a.v_h), p.read_channel, a.v_h_stride, a, p, t1 - 1, tile_rows);
    const char* x = row_pointer<T>(static_cast<const char*>(a.x), p.read_channel, a.x_stride, a, p, t1 - 1, tile_rows);
    const char* gate = row_pointer<T>(static_cast<const char*>(a.gate), SHARED ? p.head : p.read_channel, a.gate_stride, a, p, t1 - 1, tile_rows);
    const unsigned s_ring = (unsigned)__cvta_generic_to_shared(s_raw) + threadIdx.x * (FLAT ? 1 : V) * sizeof(T);
    const int groups = a.groups;
    const long long row_first = (long long)p.chain * a.chain_rows + (long long)(t1 - 1) * tile_rows + p.row0;
    const bool want_x = APPLY && a.v_x && p.active, want_gate = APPLY && a.v_gate && !SHARED && p.active;
    char* to_x = row_pointer<T>(static_cast<char*>(a.v_x), p.channel, a.h_stride, a, p, t1 - 1, tile_rows);
    char* to_gate = row_pointer<T>(static_cast<char*>(a.v_gate), SHARED ? p.head : p.channel, a.gate_out_stride, a, p, t1 - 1, tile_rows);
    float* to_part = a.gate_parts + ((a.reverse ? a.rows - 1 - row_first : row_first) + (long long)p.part * a.rows) * a.gate_heads + p.head;
    const int part_stride = a.reverse ? -a.gate_heads : a.gate_heads;
    const float* from_start = a.checkpoints + (((long long)p.chain * a.tiles + t1 - 1) * groups + p.group) * a.channels + p.read_channel;

    float q_carry[V], start[V], start_next[V];
    Map<V, A> all;
    identity(all);
    if (APPLY) carry_of_segment<false>(a, p, sh[0], q_carry);
    Borders<false, L> borders;
    borders.begin(a, p.chain, (t1 - 1) * tile_rows, reinterpret_cast<int*>(s_zeros + (a.v_h ? 0 : kTensor)), V, p.block_head, p.part);
    T gate_now[L], gate_next[L];
    int fetched = 0;       // as in the forward
    auto fetch = [&](int t) {
        int kind = kEmpty;
        if (t >= t0) {
            kind = borders.prepare(a, t, t * tile_rows);
            if (kind != kEmpty) {
                const unsigned to = s_ring + fetched * stage_bytes;
                if constexpr (FLAT) {
                    const FlatPiece piece(a, p, t * tile_rows, tile_rows, a.h_stride);
                    if (a.v_h) fetch_flat<L>(to + kVhAt * kTensor, static_cast<const char*>(a.v_h), piece);
                    if (!SHARED) fetch_flat<L>(to + kGateAt * kTensor, static_cast<const char*>(a.gate), piece);
                    if (APPLY) fetch_flat<L>(to + kXAt * kTensor, static_cast<const char*>(a.x), piece);
                } else {
                    const int rest = a.chain_rows - t * tile_rows;
                    const int left = min(rest - p.row0, L);
                    if constexpr (V * sizeof(T) == 2) {
                        NarrowRows<T, L> rx, rg, rv;
                        if (a.v_h) rv.load(vh, a.v_h_stride, left);
                        if (!SHARED) rg.load(gate, a.gate_stride, left);
                        if (APPLY) rx.load(x, a.x_stride, left);
                        unsigned char* at = s_raw + fetched * stage_bytes;
                        if (a.v_h) rv.store(at + kVhAt * kTensor);
                        if (!SHARED) rg.store(at + kGateAt * kTensor);
                        if (APPLY) rx.store(at + kXAt * kTensor);
                    } else {
                        if (a.v_h) fetch_rows<T, V, L>(to + kVhAt * kTensor, vh, a.v_h_stride, rest >= tile_rows, left, static_cast<const char*>(a.v_h));
                        if (!SHARED) fetch_rows<T, V, L>(to + kGateAt * kTensor, gate, a.gate_stride, rest >= tile_rows, left, static_cast<const char*>(a.gate));
                        if (APPLY) fetch_rows<T, V, L>(to + kXAt * kTensor, x, a.x_stride, rest >= tile_rows, left, static_cast<const char*>(a.x));
                    }
                }
            }
            vh -= a.v_h_step;
            x -= a.x_step;
            if (!SHARED) gate -= a.gate_step;
        }
        fetched = fetched + 1 == STAGES ? 0 : fetched + 1;
        copies_issued();
        return kind;
    };
    // what goes through registers: one tile ahead
    auto fetch_next = [&](int t) {
        if (SHARED) {
            fetch_shared_gates<T, L>(gate_next, gate, a.gate_stride, t >= t0 ? min(a.chain_rows - t * tile_rows - p.row0, L) : 0);
            gate -= a.gate_step;
        }
        if (APPLY && t >= t0) {
            const Pack<float, V> pack = load_pack<float, V>(from_start);
#pragma unroll
            for (int v = 0; v < V; ++v) start_next[v] = pack.e[v];
            from_start -= (long long)groups * a.channels;
        }
    };
    if (!a.v_h) {
        for (unsigned i = threadIdx.x * 4; i < kTensor; i += kWalkThreads * 4) *reinterpret_cast<unsigned*>(s_zeros + i) = 0;
    }
    int kind = fetch(t1 - 1), kind_next = kEmpty, written = -1;   // written: a flat tile whose results wait in shared memory
    fetch_next(t1 - 1);
    if (FLAT) copies_landed<0>();
    __syncthreads();
    int stage = 0, stage_written = 0;
    auto write_back = [&] {
        if (written >= 0) {
            const FlatPiece piece(a, p, written * tile_rows, tile_rows, a.h_stride);
            const float* from = reinterpret_cast<const float*>(s_raw + stage_written * stage_bytes);
            if (a.v_x) write_flat<L>(static_cast<char*>(a.v_x), piece, from + kXAt * (L * kWalkThreads * V));
            if (a.v_gate && !SHARED) write_flat<L>(static_cast<char*>(a.v_gate), piece, from + kGateAt * (L * kWalkThreads * V));
        }
        written = -1;
    };
    for (int t = t1 - 1; t >= t0; --t, kind = kind_next, stage = stage + 1 == STAGES ? 0 : stage + 1, to_x -= a.h_step,
             to_gate -= a.gate_out_step, to_part -= (long long)tile_rows * part_stride) {
        const int p0 = t * tile_rows;
        if (SHARED) {
#pragma unroll
            for (int l = 0; l < L; ++l) gate_now[l] = gate_next[l];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) start[v] = start_next[v];
        fetch_next(t - 1);
        kind_next = fetch(t - 1);
        if (!FLAT) copies_landed<1>();
        const int left = min(a.chain_rows - p0 - p.row0, L);
        // a shared gate's sum over this block's channels
        auto store_gate_sum = [&](int l, float sum) {
            if (a.parts == 1) from_float(sum, *reinterpret_cast<T*>(to_gate + l * a.gate_out_stride));
            else to_part[(long long)l * part_stride] = sum;
        };
        if (kind == kEmpty) {
            if constexpr (FLAT) {
                const FlatPiece piece(a, p, p0, tile_rows, a.h_stride);
                if (APPLY && a.v_x) write_flat<L>(static_cast<char*>(a.v_x), piece, nullptr);
                if (APPLY && a.v_gate && !SHARED) write_flat<L>(static_cast<char*>(a.v_gate), piece, nullptr);
                copies_landed<0>();
            } else {
                if (want_x) store_zero_rows<T, V, L>(to_x, a.h_stride, left);
                if (want_gate) store_zero_rows<T, V, L>(to_gate, a.gate_out_stride, left);
            }
            if (APPLY && SHARED && a.v_gate && p.leads)
                for (int l = 0; l < left; ++l) store_gate_sum(l, 0.f);
            __syncthreads();
            if (FLAT) {
                write_back();
                __syncthreads();    // before its stage is filled again
            }
            continue;
        }
        const FlatPiece piece(a, p, p0, tile_rows, a.h_stride);
        auto row_at = [&](int k, int l) {      // as in the forward
            unsigned char* base = k == kVhAt && !a.v_h ? s_zeros : s_raw + stage * stage_bytes + k * kTensor;
            return reinterpret_cast<T*>(base) + (FLAT ? max(piece.row(a, p.row0 + l), 0) : l * kWalkThreads + (int)threadIdx.x) * V;
        };
        auto tile = [&](auto plain) {
            constexpr bool PLAIN = decltype(plain)::value;
            const RowBorders<PLAIN> rows(borders.table(t), p);
            float m[L][A], u[L][V];
            Map<V, A> own;
            identity(own);
            BorderStates<false, V> ends(p.active ? a.v_state_out : nullptr, rows.end, rows.end_id, a.channels, p.channel);
#pragma unroll
            for (int l = L - 1; l >= 0; --l) {
                const bool outside = rows.is_outside(l);
                Pack<T, A> g;
                if (SHARED) g.e[0] = gate_now[l];
                else g = load_pack<T, A>(row_at(kGateAt, l));
                const Pack<T, V> d = load_pack<T, V>(row_at(kVhAt, l));
                if (rows.ends(l)) {
                    ends.take(own.b);
                    own.closed = 1;
                }
                float f[A], dv[V];
                gate_registers<T, LOGIT>(g, m[l]);
                gate_f<LOGIT>(m[l], f);
#pragma unroll
                for (int v = 0; v < V; ++v) dv[v] = outside ? 0.f : to_float(d.e[v]);
                if (outside) {
#pragma unroll
                    for (int v = 0; v < A; ++v) f[v] = 1.f;
                }
                mul(own.a, f, own.a);
                add(own.b, dv, own.b);
                mul(own.b, f, own.b);
            }
            const Map<V, A> after = publish_map<false, PLAIN>(a, p, own, sh[t & 1]);
            if (FLAT) copies_landed<0>();
            __syncthreads();
            if (FLAT) write_back();
            if (!APPLY) {
                pass_entries<false, PLAIN>(a, p, sh[t & 1], all);
                return;
            }
            pass_entries<false, PLAIN>(a, p, sh[t & 1], q_carry);
            {   // u_t: h_{t-1}, coupled: h_{t-1} - x_t.  Worked out while the first threads carry q through the tile's maps.
                float h[V];
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = start[v];
                BorderStates<true, V> begins(p.active ? a.state_in : nullptr, rows.first, rows.first_id, a.channels, p.channel);
#pragma unroll
                for (int l = 0; l < L; ++l) {
                    if (rows.begins(l)) begins.take(h);
                    const Pack<T, V> xl = load_pack<T, V>(row_at(kXAt, l));
                    float f[A], k[A], xv[V], n[V];
                    gate_f<LOGIT>(m[l], f);
#pragma unroll
                    for (int v = 0; v < V; ++v) xv[v] = to_float(xl.e[v]);
                    if (COUPLED) {
                        const float minus[1] = {-1.f};
                        mul_add(u[l], minus, xv, h);
                        gate_k<LOGIT>(m[l], f, k);
                        mul(xv, k, xv);
                    } else {
#pragma unroll
                        for (int v = 0; v < V; ++v) u[l][v] = h[v];
                    }
                    mul_add(n, f, h, xv);
#pragma unroll
                    for (int v = 0; v < V; ++v) h[v] = rows.is_outside(l) ? h[v] : n[v];
                }
            }
            __syncthreads();
            float q[V];
            entry_state(a, p, sh[t & 1], q);
            if (a.shuffle) apply_map<PLAIN>(q, after);
            [[maybe_unused]] char *row_x = to_x + (L - 1) * a.h_stride, *row_gate = to_gate + (L - 1) * a.gate_out_stride;
            BorderStates<false, V> again(p.active ? a.v_state_out : nullptr, rows.end, rows.end_id, a.channels, p.channel);
#pragma unroll
            for (int l = L - 1; l >= 0; --l) {
                const bool outside = rows.is_outside(l);
                if (rows.ends(l)) again.take(q);
                const Pack<T, V> d = load_pack<T, V>(row_at(kVhAt, l));
                float f[A], k[A], slope[A], dx[V], dg[V], g[V], n[V], sum = 0.f;
                gate_f<LOGIT>(m[l], f);
                gate_k<LOGIT>(m[l], f, k);
                if (LOGIT) mul(slope, f, k);
                else slope[0] = 1.f;
#pragma unroll
                for (int v = 0; v < V; ++v) g[v] = outside ? 0.f : to_float(d.e[v]);
                add(g, g, q);
                if (COUPLED) {
                    mul(dx, k, g);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) dx[v] = g[v];
                }
                mul(dg, g, u[l]);
                if (!SHARED && LOGIT) mul(dg, slope, dg);
                mul(n, f, g);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    dx[v] = outside ? 0.f : dx[v];
                    dg[v] = outside ? 0.f : dg[v];
                    if (SHARED) sum += dg[v];
                    q[v] = outside ? q[v] : n[v];
                }
                if constexpr (FLAT) {
                    store_floats_if<T, V>(row_at(kXAt, l), dx, want_x && (PLAIN || l < left));
                } else {
                    store_floats_if<T, V>(reinterpret_cast<T*>(row_x), dx, want_x && (PLAIN || l < left));
                    row_x -= a.h_stride;
                }
                if (rows.begins(l) && p.active && a.v_state_in)
                    store_floats<float, V>(a.v_state_in + (long long)rows.first_id[l] * a.channels + p.channel, q);
                if (!SHARED) {
                    if constexpr (FLAT) {
                        store_floats_if<T, V>(row_at(kGateAt, l), dg, want_gate && (PLAIN || l < left));
                    } else {
                        store_floats_if<T, V>(reinterpret_cast<T*>(row_gate), dg, want_gate && (PLAIN || l < left));
                        row_gate -= a.gate_out_stride;
                    }
                } else if (a.v_gate) {
                    sum = p.active && !outside ? sum * slope[0] : 0.f;   // whatever lies in the gates of rows outside
                    for (int off = a.head_threads >> 1; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                    if (p.leads && (PLAIN || l < left)) store_gate_sum(l, sum);
                }
            }
        };
        if (kind == kPlain) tile(std::true_type{});
        else tile(std::false_type{});
        if (FLAT && APPLY) {
            written = t;
            stage_written = stage;
        }
    }
    if (FLAT) {
        __syncthreads();
        write_back();
    }
    if (APPLY) pass_empty_sequences(a, a.v_state_out, a.v_state_in);
    else store_segment_map(a, p, all);
}

// ---- launches: one source file per storage type and direction instantiates these ------------------------------------------
template <typename T, int V, bool FORWARD, bool LOGIT, bool COUPLED, bool SHARED, bool APPLY>
int launch_walk(const RecurrenceLaunch& c, cudaStream_t s) {
    constexpr int L = walk_rows<T>(V);
    auto kernel = [] {
        if constexpr (FORWARD) return recurrence_forward_kernel<T, V, LOGIT, COUPLED, SHARED, APPLY>;
        else return recurrence_backward_kernel<T, V, LOGIT, COUPLED, SHARED, APPLY>;
    }();
    const int tensors = FORWARD ? (SHARED ? 1 : 2) : (APPLY ? 1 : 0) + (SHARED ? 0 : 1) + (c.args.v_h ? 1 : 0);
    const size_t smem = (walk_stages(V) * tensors + (!FORWARD && !c.args.v_h ? 1 : 0)) * walk_tensor_bytes<T>(V) + kTables * sizeof(int) * table_ints(c.args.groups, L);
    {   // more than 48 KB with the static part, for most calls: asked for once per device
        static std::atomic<u64> asked{0};
        int device = 0;
        DSB_CUDA_CHECK(cudaGetDevice(&device));
        const u64 bit = device < 64 ? 1ull << device : 0;
        if (!bit || !(asked.load(std::memory_order_relaxed) & bit)) {
            DSB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024));
            asked.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    kernel<<<c.blocks, kWalkThreads, smem, s>>>(c.args);
    DSB_LAUNCH_CHECK();
    return DSB_OK;
}
template <typename T, int V, bool FORWARD, bool LOGIT, bool COUPLED, bool SHARED>
int run_walk(const RecurrenceLaunch& c, cudaStream_t s) {
    if (c.args.segments > 1) {
        const int rc = launch_walk<T, V, FORWARD, LOGIT, COUPLED, SHARED, false>(c, s);
        if (rc != DSB_OK) return rc;
    }
    return launch_walk<T, V, FORWARD, LOGIT, COUPLED, SHARED, true>(c, s);
}
template <typename T, int V, bool FORWARD, bool LOGIT, bool COUPLED>
int run_walk(const RecurrenceLaunch& c, cudaStream_t s) {
    return c.args.shared ? run_walk<T, V, FORWARD, LOGIT, COUPLED, true>(c, s) : run_walk<T, V, FORWARD, LOGIT, COUPLED, false>(c, s);
}
template <typename T, int V, bool FORWARD>
int run_walk(const RecurrenceLaunch& c, cudaStream_t s) {
    if (c.args.logit)
        return c.args.coupled ? run_walk<T, V, FORWARD, true, true>(c, s) : run_walk<T, V, FORWARD, true, false>(c, s);
    return c.args.coupled ? run_walk<T, V, FORWARD, false, true>(c, s) : run_walk<T, V, FORWARD, false, false>(c, s);
}
template <typename T, bool FORWARD>
int run_walk(const RecurrenceLaunch& c, cudaStream_t s) {
    if constexpr (sizeof(T) == 4)
        if (c.vec == 3) return run_walk<T, 3, FORWARD>(c, s);
    if (c.vec == 2) return run_walk<T, 2, FORWARD>(c, s);
    return c.vec == 4 ? run_walk<T, 4, FORWARD>(c, s) : run_walk<T, 1, FORWARD>(c, s);
}

}  // namespace dsb
