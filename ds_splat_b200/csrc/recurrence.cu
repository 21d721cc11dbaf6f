// Gated linear recurrence over sequences, forward and backward, and its single-row form:
//     f_t = gate_t or 1 / (1 + exp(-gate_t)),   h_t = f_t h_{t-1} + i_t,   i_t = x_t or, coupled, (1 - f_t) x_t
//     g_t = v_h_t + q_{t+1},   q_t = f_t g_t,   v_x_t = g_t or (1 - f_t) g_t
//     v_f_t = sum over the channels that share the gate of g_t (h_{t-1}, coupled: h_{t-1} - x_t),   v_state_in = q_0
// Not part of the reference as an operator of its own; its blend (cpp/rasterizer_kernels.cu:341-431) is the coupled form
// over a tile's list, back to front, with f = 1 - alpha.
//
// recurrence.cuh holds the kernels that walk along sequences, recurrence_<direction>_<type>.cu instantiate them; here are the
// single-row kernel, the argument checks and the rules by which a call is cut into blocks.
#include <cmath>

#include "recurrence.cuh"

namespace dsb {

template <> int run_recurrence_forward<float>(const RecurrenceLaunch&, cudaStream_t);
template <> int run_recurrence_forward<__half>(const RecurrenceLaunch&, cudaStream_t);
template <> int run_recurrence_forward<__nv_bfloat16>(const RecurrenceLaunch&, cudaStream_t);
template <> int run_recurrence_backward<float>(const RecurrenceLaunch&, cudaStream_t);
template <> int run_recurrence_backward<__half>(const RecurrenceLaunch&, cudaStream_t);
template <> int run_recurrence_backward<__nv_bfloat16>(const RecurrenceLaunch&, cudaStream_t);

namespace {

constexpr long long kMaxRows = (1ll << 31) - (1 << 16);   // positions are 32-bit, the last tile's end included
constexpr int kMaxChannels = (int)kMaxRows;               // and so are channels, with those of threads beyond the last
constexpr long long kMaxBlocks = (1ll << 31) - 1;

// v_gate = sum of the channel blocks' shares of it, in their order
template <typename T>
__global__ void __launch_bounds__(kWalkThreads) recurrence_gate_sum_kernel(const float* parts, int count, long long n, T* v_gate) {
    for (long long i = (long long)blockIdx.x * kWalkThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kWalkThreads) {
        float sum = 0.f;
        for (int k = 0; k < count; ++k) sum += parts[k * n + i];
        from_float(sum, v_gate[i]);
    }
}

template <typename T, int V, bool LOGIT>
__global__ void __launch_bounds__(kWalkThreads)
recurrence_step_kernel(const T* x, const T* gate, float* state, T* h, const long long count, const int channels, const int per_head,
                       const long long x_stride, const long long gate_stride, const int coupled) {
    const long long i = ((long long)blockIdx.x * kWalkThreads + threadIdx.x) * V;
    if (i >= count) return;
    const long long s = i / channels;
    const int c = (int)(i - s * channels);
    const Pack<T, V> px = load_pack<T, V>(x + s * x_stride + c);
    const Pack<float, V> ps = load_pack<float, V>(state + i);
    float o[V], f = 0.f, k = 0.f;
    auto take = [&](T g) {
        Pack<T, 1> one;
        one.e[0] = g;
        float e1[1], f1[1], k1[1];
        gate_registers<T, LOGIT>(one, e1);
        gate_f<LOGIT>(e1, f1);
        gate_k<LOGIT>(e1, f1, k1);
        f = f1[0];
        k = k1[0];
    };
    Pack<T, V> pg;
    if (per_head > 1) take(gate[s * gate_stride + c / per_head]);
    else pg = load_pack<T, V>(gate + s * gate_stride + c);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (per_head == 1) take(pg.e[v]);
        const float xv = to_float(px.e[v]);
        o[v] = fmaf(f, ps.e[v], coupled ? k * xv : xv);
    }
    store_floats<float, V>(state + i, o);
    store_floats<T, V>(h + i, o);
}

// ---- host ----------------------------------------------------------------------------------------------------------------

struct Layout {            // how a call is cut; the same for the forward and the backward of one shape
    int vec;               // channels per thread: 4, 3, 2 or 1
    int tx, groups;        // threads side by side on one row; groups of rows in a tile
    bool shuffle;
    int per_head;          // channels that share a gate; all of them when every channel has its own
    int head_blocks;       // blocks side by side, without the parts; 1 when every channel has its own gate
    int block_heads;       // heads of a block
    int parts;             // channel blocks per head
    bool table;            // one chain over all rows, with sequence borders anywhere; else one chain per sequence
    int tile_rows;
    int64_t chains, chain_rows, tiles;     // tiles of a chain
    int64_t segments, segment_tiles;       // of a chain
};
// Two blocks are what registers allow an SM, and shared memory too but for some calls with one thread a row, whose 256 groups make
// large border tables: a single 32-bit channel (81 KB of tables; 36 to 72 KB of stages in the backward, 48 in the forward with a
// gate of its own) and three with gates of their own (39 KB; 90 and 135 KB of stages).  Those run one block an SM, and where they
// are cut, twice the segments that run at once.
constexpr int kSms = 148, kBlocksPerSm = 2;
// A chain of fewer tiles is not cut: a tile after another takes a block about 2 us, a second launch and its first tile 6 us.
constexpr int kLeastTilesToCut = 8;

int check_shape(const DsbRecurrence& s, bool step) {
    DSB_REQUIRE(s.dtype == DSB_DTYPE_F32 || s.dtype == DSB_DTYPE_F16 || s.dtype == DSB_DTYPE_BF16, "recurrence: unknown dtype %d", s.dtype);
    DSB_REQUIRE(s.gate_form == DSB_GATE_DECAY || s.gate_form == DSB_GATE_LOGIT, "recurrence: unknown gate form %d", s.gate_form);
    DSB_REQUIRE(s.channels >= 1 && s.gate_heads >= 1 && s.channels % s.gate_heads == 0,
                "recurrence: %d channels do not split into %d gate heads", s.channels, s.gate_heads);
    DSB_REQUIRE(s.channels <= kMaxChannels, "recurrence: at most 2^31 - 2^16 channels, got %d", s.channels);
    DSB_REQUIRE(s.rows >= 0 && s.rows <= kMaxRows, "recurrence: at most 2^31 - 2^16 rows, got %lld", (long long)s.rows);
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
    // colours: contiguous rows of three 32-bit channels are taken flat
    if (s.channels == 3 && s.dtype == DSB_DTYPE_F32 && s.x_stride == 3 && (shared || s.gate_stride == 3)) return 3;
    const int together = shared ? s.channels / s.gate_heads : s.channels;
    return together % 4 == 0 ? 4 : together % 2 == 0 ? 2 : 1;
}
Layout layout_of(const DsbRecurrence& s) {
    Layout l = {};
    if (s.rows == 0) return l;
    l.vec = shape_vec(s);
    const bool shared = s.gate_heads != s.channels;
    l.head_blocks = shared ? s.gate_heads : 1;
    l.block_heads = 1;
    l.per_head = s.channels / l.head_blocks;
    const int wide = (l.per_head + l.vec - 1) / l.vec;
    const int rows = s.dtype == DSB_DTYPE_F32 ? walk_rows<float>(l.vec) : walk_rows<__half>(l.vec);
    const int piece = l.vec * dtype_bytes(s.dtype);
    auto fill_in = [&](int tx) {
        Layout c = l;
        c.tx = tx;
        c.shuffle = tx <= 8;
        c.groups = kWalkThreads / tx;
        c.parts = (wide + tx - 1) / tx;
        c.tile_rows = c.groups * rows;
        // A chain per sequence wastes half a tile per sequence on average; a table costs a look at every row.
        c.table = s.sequence_rows == 0 || s.sequence_rows < c.tile_rows;
        c.chains = c.table ? 1 : s.sequences;
        c.chain_rows = c.table ? s.rows : s.sequence_rows;
        c.tiles = (c.chain_rows + c.tile_rows - 1) / c.tile_rows;
        c.segments = 1;
        return c;
    };
    Layout best = {};
    if (wide <= 8) {   // vec 3 among them: one thread per row
        // Narrow heads lie side by side in a block: a head alone in one would read a sector a row for a few bytes (29 x 3642 rows
        // of 112 fp16 heads of 3 channels, a training pass: 670 us then, 401 so).  As many as a row's piece needs to fill a line
        // of 128 bytes while eight threads a row are enough, so that warps compose their maps by themselves; with more threads,
        // two sectors have to do.  On the device, 8 x 4096 x 1024: 64 bf16 heads of 16 at 32 / 64 / 128 bytes, which takes 4 / 8 /
        // 16 threads, 170 / 121 / 170 us; 128 fp32 heads of 8 at 32 / 64 / 128 bytes, 2 / 4 / 8 threads, 301 / 205 / 164.
        int tx = 1;
        while (tx < wide) tx *= 2;
        while (shared && tx <= 16 && l.block_heads < s.gate_heads &&
               l.block_heads * l.per_head * dtype_bytes(s.dtype) < (tx < 8 ? 128 : 64)) {
            l.block_heads *= 2;
            tx *= 2;
        }
        l.head_blocks = (l.head_blocks + l.block_heads - 1) / l.block_heads;
        best = fill_in(tx);
        const int64_t blocks = best.chains * best.head_blocks;
        if (2 * blocks < kSms * kBlocksPerSm && best.tiles >= kLeastTilesToCut) best.segments = kSms * kBlocksPerSm / blocks;
    } else {
        // The number of threads that share a row, and whether sequences are cut (which reads the inputs twice), by what share
        // of the threads' time goes into elements: threads without channels, SMs without their two blocks, pieces of a row that
        // end inside a 32-byte sector, and the composition of a tile's maps (20 instructions an element; 60 and 9 per
        // group of rows for a thread's part of a tile) all take from it.  A shared gate's sum over its channels takes a
        // power of two of threads.
        double most = 0;
        for (int lanes = 9; lanes <= 64; ++lanes) {
            const int parts = (wide + lanes - 1) / lanes, tx = shared ? lanes : (wide + parts - 1) / parts;
            if (tx < 9 || (shared && lanes != 16 && lanes != 32)) continue;
            Layout c = fill_in(tx);
            const double elements = 20.0 * rows * l.vec;
            double share = (double)wide / (c.parts * tx) * (c.groups * tx) / kWalkThreads * elements / (elements + 60 + 9 * c.groups);
            if (c.parts > 1 && tx * piece % 32 != 0) share *= 0.93;
            const double per_sm = (double)(c.chains * c.head_blocks * c.parts) / kSms;
            const double whole = share * (per_sm <= 1 ? 0.65 * per_sm : per_sm / (kBlocksPerSm * std::ceil(per_sm / kBlocksPerSm)));
            int64_t segments = (int64_t)(kBlocksPerSm / per_sm);
            if (segments > c.tiles) segments = c.tiles;
            const double cut = segments > 1 && c.tiles >= kLeastTilesToCut ? share * per_sm * segments / kBlocksPerSm / 1.6 : 0;
            if (whole > most) { most = whole; best = c; }
            if (cut > most) { most = cut; best = c; best.segments = segments; }
        }
    }
    if (best.segments > best.tiles) best.segments = best.tiles;
    if (best.tiles > 0) {
        best.segment_tiles = (best.tiles + best.segments - 1) / best.segments;
        best.segments = (best.tiles + best.segment_tiles - 1) / best.segment_tiles;   // none of them empty
    }
    return best;
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

struct Cut { Layout layout; RecurrenceLaunch launch; };

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
    RecurrenceArgs& a = c.launch.args;
    a = RecurrenceArgs{};
    a.rows = (int)s.rows; a.chain_rows = (int)l.chain_rows; a.chains = (int)l.chains;
    a.tiles = (int)l.tiles; a.segments = (int)l.segments; a.segment_tiles = (int)l.segment_tiles;
    a.checkpoints = checkpoints;
    a.sequences = s.sequences; a.sequence_rows = s.sequence_rows; a.channels = s.channels; a.gate_heads = s.gate_heads;
    a.per_head = l.per_head; a.head_blocks = l.head_blocks; a.block_heads = l.block_heads; a.head_threads = l.tx / l.block_heads;
    a.parts = l.parts;
    a.tx = l.tx; a.groups = l.groups; a.shuffle = l.shuffle; a.entries = l.shuffle ? kWalkWarps : l.groups;
    a.logit = s.gate_form == DSB_GATE_LOGIT; a.coupled = s.coupled != 0; a.reverse = s.reverse != 0;
    a.shared = s.gate_heads != s.channels; a.table = l.table;
    a.offsets = s.offsets; a.lengths = s.lengths;
    const int64_t sign = (a.reverse ? -1 : 1) * dtype_bytes(s.dtype);
    a.x_stride = sign * s.x_stride; a.gate_stride = sign * s.gate_stride;
    a.h_stride = sign * s.channels; a.gate_out_stride = sign * s.gate_heads;
    a.x_step = l.tile_rows * a.x_stride; a.gate_step = l.tile_rows * a.gate_stride;
    a.h_step = l.tile_rows * a.h_stride; a.gate_out_step = l.tile_rows * a.gate_out_stride;
    unsigned char* w = static_cast<unsigned char*>(workspace);
    if (l.segments > 1) {
        const int64_t maps = l.chains * l.segments, bytes = up16(maps * s.channels * 4);
        a.map_a = reinterpret_cast<float*>(w); w += bytes;
        a.map_b = reinterpret_cast<float*>(w); w += bytes;
        a.map_closed = reinterpret_cast<int*>(w); w += up16(maps * 4);
    }
    if (!forward && a.shared && l.parts > 1) a.gate_parts = reinterpret_cast<float*>(w);
    const int64_t blocks = l.chains * l.segments * l.head_blocks * l.parts;
    DSB_REQUIRE(blocks <= kMaxBlocks, "recurrence: too many blocks for one launch");
    c.launch.vec = l.vec; c.launch.tile_rows = l.tile_rows; c.launch.blocks = (unsigned)blocks;
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

template <bool FORWARD>
int run_direction(const DsbRecurrence& shape, const Cut& c, cudaStream_t s) {
    int rc = DSB_OK;
    with_dtype(shape.dtype, [&](auto tag) {
        typedef decltype(tag) T;
        rc = FORWARD ? run_recurrence_forward<T>(c.launch, s) : run_recurrence_backward<T>(c.launch, s);
        if (rc == DSB_OK && !FORWARD && c.launch.args.gate_parts && c.launch.args.v_gate) {
            const long long n = shape.rows * shape.gate_heads;
            T* out = static_cast<T*>(c.launch.args.v_gate);
            if (c.launch.args.reverse) out -= (shape.rows - 1) * shape.gate_heads;
            const long long blocks = (n + kWalkThreads - 1) / kWalkThreads;
            recurrence_gate_sum_kernel<T><<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), kWalkThreads, 0, s>>>(
                c.launch.args.gate_parts, c.layout.parts, n, out);
            count_launch();
            if (cudaPeekAtLastError() != cudaSuccess) { set_error("recurrence: launch failed"); rc = DSB_ERR_CUDA; }
        }
    });
    return rc;
}

// Channels that a thread takes `lanes` at a time need every row of every tensor on such a boundary.
int vector_lanes(const DsbRecurrence& s) {
    const int vec = shape_vec(s);
    return vec == 3 ? 1 : vec;
}
int check_alignment(const void* p, int64_t stride, int elem, int lanes, const char* name) {
    if (!p || lanes == 1) return DSB_OK;
    DSB_REQUIRE(aligned(p, lanes * elem) && stride % lanes == 0,
                "recurrence: with these channels %s must start on a boundary of %d elements and its rows lie a multiple of that apart",
                name, lanes);
    return DSB_OK;
}
#define DSB_TRY(expr) do { const int rc__ = (expr); if (rc__ != DSB_OK) return rc__; } while (0)

int check_inputs(const DsbRecurrence& s, const void* x, const void* gate) {
    const int lanes = vector_lanes(s), elem = dtype_bytes(s.dtype);
    DSB_TRY(check_alignment(x, s.x_stride, elem, lanes, "x"));
    return check_alignment(gate, s.gate_stride, elem, s.gate_heads == s.channels ? lanes : 1, "the gate");
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
    return l.chains * l.tiles * l.groups * s.channels * 4;
}

int launch_recurrence_forward(const DsbRecurrence& shape, const void* x, const void* gate, const float* state_in, void* h,
                              float* state_out, float* checkpoints, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
    DSB_TRY(check_shape(shape, false));
    DSB_REQUIRE(state_out || shape.sequences == 0, "recurrence: null state_out");
    if (shape.rows == 0) return pass_states(state_in, state_out, (int64_t)shape.sequences * shape.channels, s);
    DSB_REQUIRE(x && gate, "recurrence: null pointer");
    DSB_REQUIRE(!state_in || state_in != state_out, "recurrence: state_out must not be state_in");
    const int lanes = vector_lanes(shape), elem = dtype_bytes(shape.dtype);
    DSB_TRY(check_inputs(shape, x, gate));
    DSB_TRY(check_alignment(h, shape.channels, elem, lanes, "h"));
    DSB_TRY(check_alignment(state_in, shape.channels, 4, lanes, "state_in"));
    DSB_TRY(check_alignment(state_out, shape.channels, 4, lanes, "state_out"));
    Cut c;
    DSB_TRY(make_cut(shape, true, workspace, workspace_bytes, checkpoints, &c));
    const bool r = shape.reverse != 0;
    c.launch.args.x = scan_base(x, r, shape.rows, shape.x_stride, elem);
    c.launch.args.gate = scan_base(gate, r, shape.rows, shape.gate_stride, elem);
    c.launch.args.h = scan_base(h, r, shape.rows, shape.channels, elem);
    c.launch.args.state_in = state_in; c.launch.args.state_out = state_out;
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
    const int lanes = vector_lanes(shape), elem = dtype_bytes(shape.dtype);
    DSB_TRY(check_inputs(shape, x, gate));
    DSB_TRY(check_alignment(v_h, v_h_stride, elem, lanes, "v_h"));
    DSB_REQUIRE(!v_h || shape_vec(shape) != 3 || v_h_stride == 3, "recurrence: where x's rows of three channels are contiguous, v_h's must be");
    DSB_TRY(check_alignment(v_x, shape.channels, elem, lanes, "v_x"));
    DSB_TRY(check_alignment(v_gate, shape.gate_heads, elem, shape.gate_heads == shape.channels ? lanes : 1, "v_gate"));
    DSB_TRY(check_alignment(state_in, shape.channels, 4, lanes, "state_in"));
    DSB_TRY(check_alignment(v_state_out, shape.channels, 4, lanes, "v_state_out"));
    DSB_TRY(check_alignment(v_state_in, shape.channels, 4, lanes, "v_state_in"));
    Cut c;
    DSB_TRY(make_cut(shape, false, workspace, workspace_bytes, const_cast<float*>(checkpoints), &c));
    const bool r = shape.reverse != 0;
    c.launch.args.x = scan_base(x, r, shape.rows, shape.x_stride, elem);
    c.launch.args.gate = scan_base(gate, r, shape.rows, shape.gate_stride, elem);
    c.launch.args.v_h = scan_base(v_h, r, shape.rows, v_h_stride, elem);
    c.launch.args.v_h_stride = (r ? -v_h_stride : v_h_stride) * elem;
    c.launch.args.v_h_step = c.layout.tile_rows * c.launch.args.v_h_stride;
    c.launch.args.v_x = scan_base(v_x, r, shape.rows, shape.channels, elem);
    c.launch.args.v_gate = scan_base(v_gate, r, shape.rows, shape.gate_heads, elem);
    c.launch.args.state_in = state_in; c.launch.args.v_state_out = v_state_out; c.launch.args.v_state_in = v_state_in;
    return run_direction<false>(shape, c, s);
}

int launch_recurrence_step(const DsbRecurrence& shape, const void* x, const void* gate, float* state, void* h, cudaStream_t s) {
    DSB_TRY(check_shape(shape, true));
    if (shape.rows == 0) return DSB_OK;
    DSB_REQUIRE(x && gate && state && h, "recurrence: null pointer");
    const int lanes = vector_lanes(shape), elem = dtype_bytes(shape.dtype);
    DSB_TRY(check_inputs(shape, x, gate));
    DSB_TRY(check_alignment(h, shape.channels, elem, lanes, "h"));
    DSB_TRY(check_alignment(state, shape.channels, 4, lanes, "the state"));
    const long long count = shape.rows * shape.channels;
    const long long blocks = (count / lanes + kWalkThreads - 1) / kWalkThreads;
    DSB_REQUIRE(blocks <= kMaxBlocks, "recurrence: too many elements for one launch");
    const int per_head = shape.channels / shape.gate_heads;
    with_dtype(shape.dtype, [&](auto tag) {
        typedef decltype(tag) T;
        auto launch = [&](auto kernel) {
            kernel<<<(unsigned)blocks, kWalkThreads, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(gate), state, static_cast<T*>(h),
                                                             count, shape.channels, per_head, shape.x_stride, shape.gate_stride,
                                                             shape.coupled != 0);
        };
        const bool logit = shape.gate_form == DSB_GATE_LOGIT;
        if (lanes == 4 && logit) launch(recurrence_step_kernel<T, 4, true>);
        else if (lanes == 4) launch(recurrence_step_kernel<T, 4, false>);
        else if (lanes == 2 && logit) launch(recurrence_step_kernel<T, 2, true>);
        else if (lanes == 2) launch(recurrence_step_kernel<T, 2, false>);
        else if (logit) launch(recurrence_step_kernel<T, 1, true>);
        else launch(recurrence_step_kernel<T, 1, false>);
    });
    DSB_LAUNCH_CHECK();
    return DSB_OK;
}

}  // namespace dsb
