// Selective state space scan over packed utterances: the kernels, shared by the translation
// units that instantiate them (one per element type, so they compile in parallel).
//
//   d_t = softplus(dt_t + bias)       (or dt_t + bias)         per channel
//   h_t = exp(d_t A) h_{t-1} + d_t x_t B_t                     per channel and state
//   y_t = (sum_n C_t h_t + skip x_t) silu(gate_t)              per channel
//
// It is the recursion of the forward variables (hmm_generic.hip) with a diagonal transition that
// depends on the frame, and a sum in place of the logarithm's normalisation.
//
// Layout of a wave: 16 R channels times 4 S states.  Lane 16 row + col holds the states
// row S .. row S + S - 1 of the channels col R .. col R + R - 1 in registers, so that per frame it
// reads R steps and products d x (the same for the four rows) and S values each of B and C (the same for
// 16 lanes) from LDS, where the wave itself has put a tile of frames in float32; a frame's exponentials
// are R S per lane, none computed twice.  Everything that a frame needs per channel only (softplus,
// gate, the loads and stores) is dealt out by rows: row g of the wave does frame 4 i + g, so that
// nothing is computed four times either and a row's access is 16 R neighbouring channels.
// No two waves share anything: no barriers.
//
// Bound by the vector ALU: per (frame, channel, state) an exponential, two products and two multiply-adds, 9 ns of a
// SIMD per 64 of them, and about two thirds of that again for what a frame needs per channel and for LDS.  A recording
// of 24,001 frames x 512 channels x 16 states in bfloat16 takes 113 us (28 for the recursion's arithmetic alone, 20 for
// its bytes; cut into pieces it is computed twice), 96 utterances of 100 to 300 frames x 1024 channels in float16
// 104 us (44, 35), forward and backward over 64 such x 1536 channels in bfloat16 402 us (124, 66).  One channel per lane
// with all its states, which needs no sums across lanes and no LDS but for B and C, has 8 % fewer instructions but
// registers for two waves per SIMD only, and is slower (124, 142).
#pragma once
#include "frame_ops.h"

using namespace srx_frames;

constexpr int kScanSaveEvery = 8;       // frames between two saved states
constexpr int kScanTile = 16;           // frames that a wave of the forward pass puts into LDS at once
constexpr int kScanWaves = 4;           // waves of a workgroup: neighbouring channel blocks of one unit

struct ScanParams {
    // model
    const float* A;          // [channels, states]
    const float* skip;       // [channels] or NULL
    const float* bias;       // [channels] or NULL
    int softplus;
    int channels, states, groups;
    int per_group;           // channels of a group
    int group_blocks;        // channel blocks (of 16 R) of a group
    int blocks;              // of all groups
    int wide;                // R: channels of a lane
    // frames
    const int64_t* off;
    int64_t utts, frames;
    const void *x, *dt, *B, *C, *gate;
    int64_t ld_x, ld_dt, ld_B, ld_C, ld_gate;
    // units: utterances (segment == 0) or pieces of `segment` frames of them
    int64_t units, segment;
    bool ordered;
    int round;               // utterances that give every CU a workgroup
    int* order;              // [utts] utterances by falling length, or NULL: as they come (the backward pass
                             // takes the forward pass's, behind the saved states)
    int clear;               // workgroups that set the outputs' rows of no utterance to zero (0: these are left alone)
    // forward
    const float* state_in;   // [utts, channels, states] or NULL
    float* state_out;        // the same or NULL
    void* y;
    int64_t ld_y;
    float* saved;            // states before every kScanSaveEvery-th frame, in the lanes' order
    float* seg_state;        // [units, blocks, R S / 4, 64, 4]: a piece's last state from zero, then its first state
    float* seg_sum;          // [units, blocks, 16 R]: sum of a piece's steps
    // backward
    const void* dy;
    int64_t ld_dy;
    void *dx, *ddt, *dB, *dC, *dgate;
    int64_t ld_dx, ld_ddt, ld_dB, ld_dC, ld_dgate;
    float *dA, *dskip, *dbias, *dstate_in;
    const float* dstate_out;
    int64_t parts;           // waves that sum dA, dskip, dbias over their share of the units
    float* part_A;           // [parts, blocks, R S / 4, 64, 4]
    float* part_vec;         // [parts, blocks, 2, 16 R]
    float* part_bc;          // [blocks, frames, 2, 4 S]
};

// What a wave works on: frames first .. last - 1 of utterance utt, which begins at `begin`.
struct ScanUnit {
    int64_t utt, begin, first, last;
    bool head, tail;         // it has the utterance's first / last frame (an empty utterance: both)
};

// Offsets are the caller's device data: whatever they hold, no frame outside the buffers is touched.
__device__ __forceinline__ void scan_bounds(const ScanParams& p, int64_t utt, int64_t& begin, int64_t& end) {
    begin = min(max(p.off[utt], (int64_t)0), p.frames);
    end = min(max(p.off[utt + 1], begin), p.frames);
}

__device__ __forceinline__ bool scan_unit(const ScanParams& p, int64_t unit, ScanUnit& w) {
    int64_t begin, end;
    if (p.segment == 0) {
        int64_t utt = unit;
        if (p.order != nullptr) {                         // odd rounds the other way round: a long one beside a short one
            const int round = (int)unit / p.round, end = min((round + 1) * p.round, (int)p.utts);
            utt = p.order[round & 1 ? end - 1 - ((int)unit - round * p.round) : unit];
        }
        if (utt < 0 || utt >= p.utts) return false;       // (the saved states were not the forward pass's)
        scan_bounds(p, utt, begin, end);
        w = {utt, begin, begin, end, true, true};
        return true;
    }
    // pieces are numbered off / segment + utterance + piece: no two alike, and the utterance is
    // the last one whose first piece is not behind the number
    int64_t lo = 0, hi = p.utts - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        const int64_t at = min(max(p.off[mid], (int64_t)0), p.frames);
        if (at / p.segment + mid <= unit) lo = mid;
        else hi = mid - 1;
    }
    scan_bounds(p, lo, begin, end);
    const int64_t piece = unit - (begin / p.segment + lo);
    const int64_t first = begin + piece * p.segment;
    if (piece < 0 || (first >= end && piece > 0)) return false;
    const int64_t last = min(first + p.segment, end);
    w = {lo, begin, first, last, piece == 0, last == end};
    return true;
}

// A value that is the same in all lanes, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v);
    const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((uint64_t)v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ void uniform_unit(ScanUnit& u) {
    u.utt = uniform64(u.utt);
    u.begin = uniform64(u.begin);
    u.first = uniform64(u.first);
    u.last = uniform64(u.last);
}

// The rows of one matrix as a wave walks over them: a scalar address that moves with the frames and a
// 32-bit offset of the lane's own (its row among the first `frames` of a tile, its channel), so that a walk over
// eight matrices costs eight vector registers.  (The entry points refuse pitches that offset cannot reach.)
template <typename T>
struct ScanRows {
    GlobalChar* at;          // frame 0 of the tile
    int64_t pitch;           // bytes
    unsigned off;
    __device__ __forceinline__ ScanRows() {}
    __device__ __forceinline__ ScanRows(const void* base, int64_t ld, int64_t frame, int row, int column) {
        pitch = ld * (int64_t)sizeof(T);
        at = (GlobalChar*)const_cast<void*>(base) + frame * pitch;
        off = (unsigned)row * (unsigned)pitch + (unsigned)column * (unsigned)sizeof(T);
    }
    template <int V>
    __device__ __forceinline__ Pack<T, V> load(int more) const { return load_global<V, T>(at + more * pitch, off); }
    template <int V>
    __device__ __forceinline__ void store(int more, const Pack<T, V>& v) const { store_global<V, T>(at + more * pitch, off, v); }
    __device__ __forceinline__ void move(int frames) { at += frames * pitch; }
};

// The utterances by falling length (the same lengths in their own order): the waves of long ones start first, and the
// chip is not left waiting for one that began last; and as the first rounds of workgroups stay on their CUs side by
// side, every other round is taken backwards (scan_unit), so that the lengths of a CU's workgroups add up to much the
// same.  96 utterances of 100 to 300 frames x 1024 channels, 16 states: 117 us as they come, 107 by falling length, 96
// with the rounds; utterances of equal length pay 6 us for this launch.  Every thread
// counts the utterances before its own, in one workgroup.
constexpr int kScanOrderedLeast = 16, kScanOrdered = 1024;
static __global__ __launch_bounds__(kScanOrdered) void scan_order_kernel(ScanParams p) {
    __shared__ __align__(16) int lengths[kScanOrdered];
    const int u = threadIdx.x, n = (int)p.utts;
    int64_t begin = 0, end = 0;
    if (u < n) scan_bounds(p, u, begin, end);
    const int mine = (int)min(end - begin, (int64_t)0x7fffffff);
    lengths[u] = u < n ? mine : -1;
    __syncthreads();
    if (u >= n) return;
    int before = 0;
    for (int v = 0; v < n; v += 4) {
        const Pack<int, 4> q = load_pack<4>(lengths + v);
#pragma unroll
        for (int k = 0; k < 4; ++k) before += q.v[k] > mine || (q.v[k] == mine && v + k < u);
    }
    p.order[before] = u;
}

// Channels of a wave's block, and where they are.  QUADS false: the four rows of 16 lanes hold the four groups of
// states, lane 16 row + col; true: four neighbouring lanes do, lane 4 col + row.
template <int R, int S, bool QUADS>
struct ScanLane {
    static constexpr int kChannels = 16 * R, kStates = 4 * S;
    static_assert(R * S % 4 == 0, "states move in fours");
    int lane, row, col;
    int group, channel, left;    // first channel of this lane, how many of its R exist
    int end;                     // the group's last channel
    int state;                   // first state of this lane
    bool full;                   // the block has all its channels (the same for the whole wave)
    __device__ __forceinline__ ScanLane(const ScanParams& p, int block) {
        lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));       // (or what follows from it would wait in registers from task to task)
        row = QUADS ? lane & 3 : lane >> 4;
        col = QUADS ? lane >> 2 : lane & 15;
        group = block / p.group_blocks;
        const int first = (block - group * p.group_blocks) * kChannels, base = first + col * R;
        channel = group * p.per_group + base;
        left = min(max(p.per_group - base, 0), R);
        end = (group + 1) * p.per_group - 1;
        state = row * S;
        full = first + kChannels <= p.per_group;
    }
    __device__ __forceinline__ bool exists(const ScanParams& p, int r, int s) const { return r < left && state + s < p.states; }
    // R neighbouring values of frame 4 i + row, or of frame `last` where that is behind it.  A whole block's are one
    // access without a branch; elsewhere the group's last channel stands in for those that do not exist.
    template <typename T>
    __device__ __forceinline__ Pack<T, R> load_any(const ScanRows<T>& rows, int i, int last) const {
        int t = min(4 * i + row, last), c = channel;
        asm volatile("" : "+v"(t), "+v"(c));             // (nothing of this is worth a register in the loop)
        const T* at = (const T*)(rows.at + t * rows.pitch);
        Pack<T, R> v;
#pragma unroll
        for (int r = 0; r < R; ++r) v.v[r] = at[min(c + r, end)];
        __builtin_amdgcn_sched_barrier(0);               // (one row's addresses at a time)
        return v;
    }
    template <typename T>
    __device__ __forceinline__ void store(const ScanRows<T>& rows, int i, const Pack<T, R>& v) const {
        if (full) {
            rows.template store<R>(4 * i, v);
            return;
        }
        T* at = (T*)global_at(rows.at + 4 * i * rows.pitch, rows.off);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r < left) at[r] = v.v[r];
    }
};
// S states of frame t of a tile's B or C from state s0 on, zeros for those that do not exist and for frames behind the
// last one.
template <int S, typename T>
__device__ __forceinline__ Pack<T, S> scan_load_bc(const ScanRows<T>& rows, int t, int last, int group, int s0, int states) {
    const int there = t <= last ? states : 0;
    t = min(t, last);
    asm volatile("" : "+v"(t), "+v"(s0));
    const T* at = (const T*)(rows.at + t * rows.pitch) + (int64_t)group * states;
    Pack<T, S> v;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const T x = at[min(s0 + s, states - 1)];
        v.v[s] = s0 + s < there ? x : (T)0.0f;
    }
    __builtin_amdgcn_sched_barrier(0);
    return v;
}

template <int R, int S, bool Q>
__device__ __forceinline__ void scan_load_states(const float* from, const ScanParams& p, const ScanLane<R, S, Q>& w,
                                                 int64_t utt, float (&h)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s)
            h[r][s] = from != nullptr && r < w.left && w.state + s < p.states
                          ? from[(utt * p.channels + w.channel + r) * p.states + w.state + s] : 0.0f;
}
template <int R, int S, bool Q>
__device__ __forceinline__ void scan_store_states(float* to, const ScanParams& p, const ScanLane<R, S, Q>& w,
                                                  int64_t utt, const float (&h)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (r < w.left && w.state + s < p.states)
                to[(utt * p.channels + w.channel + r) * p.states + w.state + s] = h[r][s];
}
// The same in an order of their own, in which an instruction of the wave covers whole lines: for every four
// values of a lane, lane 16 row + col (padded channels and states included).
template <int R, int S, bool Q>
__device__ __forceinline__ void scan_load_lanes(const float* from, int64_t at, const ScanLane<R, S, Q>& w, float (&h)[R][S]) {
    const float* base = from + (at * (R * S / 4) * 64 + w.row * 16 + w.col) * 4;
#pragma unroll
    for (int q = 0; q < R * S / 4; ++q) {
        const Pack<float, 4> v = load_pack<4>(base + q * 256);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[(q * 4 + k) / S][(q * 4 + k) % S] = v.v[k];
    }
}
template <int R, int S, bool Q>
__device__ __forceinline__ void scan_store_lanes(float* to, int64_t at, const ScanLane<R, S, Q>& w, const float (&h)[R][S]) {
    float* base = to + (at * (R * S / 4) * 64 + w.row * 16 + w.col) * 4;
#pragma unroll
    for (int q = 0; q < R * S / 4; ++q) {
        Pack<float, 4> v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v.v[k] = h[(q * 4 + k) / S][(q * 4 + k) % S];
        store_pack(base + q * 256, v);
    }
}
// Zeros in the place of what does not exist.
template <int R, int S, bool Q>
__device__ __forceinline__ void scan_clear_absent(const ScanParams& p, const ScanLane<R, S, Q>& w, float (&h)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s) h[r][s] = w.exists(p, r, s) ? h[r][s] : 0.0f;
}
__device__ __forceinline__ int64_t scan_slot(const ScanUnit& u, int64_t t) {
    return u.begin / kScanSaveEvery + u.utt + (t - u.begin) / kScanSaveEvery;
}

// An infinite rate of decay becomes the largest number, so that a step of zero (which the frames behind an utterance's
// end have) leaves a state alone, as it does for any A.
__device__ __forceinline__ float scan_finite(float v) { return fabsf(v) > 3.4028234e38f ? copysignf(3.4028234e38f, v) : v; }
// A log2(e), so that the decay is one product and the hardware's 2^x.
__device__ __forceinline__ float scan_log2_decay(float a) { return scan_finite(a * 1.44269504088896341f); }
template <int R, int S, bool Q>
__device__ __forceinline__ void scan_load_A(const ScanParams& p, const ScanLane<R, S, Q>& w, float (&A2)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s)
            A2[r][s] = r < w.left && w.state + s < p.states
                           ? scan_log2_decay(p.A[(int64_t)(w.channel + r) * p.states + w.state + s]) : 0.0f;
}

// ---- forward ------------------------------------------------------------------------------

// A tile of frames on its way from memory: row g of the wave has frames 4 i + g.  Addresses advance with the tiles.
template <typename T, int R, int S, bool GATE, bool WITH_Y>
struct ScanTileRaw {
    Pack<T, R> x[4], dt[4], z[4];
    Pack<T, S> b, c;
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            arrive(x[i]);
            arrive(dt[i]);
            if (GATE && WITH_Y) arrive(z[i]);
        }
        arrive(b);
        if (WITH_Y) arrive(c);
    }
};
template <typename T, int R, int S, bool GATE, bool WITH_Y>
struct ScanTileReader {
    ScanRows<T> x, dt, z, b, c;
    bool all_states;
    __device__ __forceinline__ ScanTileReader(const ScanParams& p, const ScanLane<R, S, false>& w, int64_t first) {
        const int s0 = w.group * p.states + (w.lane & 3) * S;
        x = ScanRows<T>(p.x, p.ld_x, first, w.row, w.channel);
        dt = ScanRows<T>(p.dt, p.ld_dt, first, w.row, w.channel);
        if (GATE && WITH_Y) z = ScanRows<T>(p.gate, p.ld_gate, first, w.row, w.channel);
        b = ScanRows<T>(p.B, p.ld_B, first, w.lane >> 2, s0);
        if (WITH_Y) c = ScanRows<T>(p.C, p.ld_C, first, w.lane >> 2, s0);
        all_states = p.states == 4 * S;
    }
    // The next `frames` frames (at least one): a whole tile without a branch, a shorter one with its last frame in
    // place of those behind it, which are not used.
    __device__ __forceinline__ void next(const ScanParams& p, const ScanLane<R, S, false>& w, int64_t frames,
                                         ScanTileRaw<T, R, S, GATE, WITH_Y>& to) {
        const int last = (int)min(frames, (int64_t)kScanTile) - 1;
        if (last == kScanTile - 1 && w.full) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                to.x[i] = x.template load<R>(4 * i);
                to.dt[i] = dt.template load<R>(4 * i);
                if (GATE && WITH_Y) to.z[i] = z.template load<R>(4 * i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                to.x[i] = w.load_any(x, i, last);
                to.dt[i] = w.load_any(dt, i, last);
                if (GATE && WITH_Y) to.z[i] = w.load_any(z, i, last);
            }
        }
        if (last == kScanTile - 1 && all_states) {
            to.b = b.template load<S>(0);
            if (WITH_Y) to.c = c.template load<S>(0);
        } else {
            const int s0 = (w.lane & 3) * S;
            to.b = scan_load_bc<S>(b, w.lane >> 2, last, w.group, s0, p.states);
            if (WITH_Y) to.c = scan_load_bc<S>(c, w.lane >> 2, last, w.group, s0, p.states);
        }
        x.move(kScanTile);
        dt.move(kScanTile);
        if (GATE && WITH_Y) z.move(kScanTile);
        b.move(kScanTile);
        if (WITH_Y) c.move(kScanTile);
    }
};

// A frame's values for one lane, from the wave's LDS.
template <int R, int S>
struct ScanFrame {
    Pack<float, R> d, du, q;
    Pack<float, S> b, c;
    template <bool WITH_B, bool WITH_C, bool QUADS>
    __device__ __forceinline__ void load(const ScanLane<R, S, QUADS>& w, int j, const float* sD, const float* sU,
                                         const float* sP, const float* sB, const float* sC) {
        d = load_pack<R>(sD + j * (16 * R) + w.col * R);
        if (sU != nullptr) du = load_pack<R>(sU + j * (16 * R) + w.col * R);
        if (sP != nullptr) q = load_pack<R>(sP + j * (16 * R) + w.col * R);
        if (WITH_B) b = load_pack<S>(sB + j * (4 * S) + w.state);
        if (WITH_C) c = load_pack<S>(sC + j * (4 * S) + w.state);
    }
};

// MODE 0: the outputs.  MODE 1: only the last state of a piece and the sum of its steps.
// Four waves per SIMD where their registers hold it with a few spilled outside the loop (16 states in float32, 128
// utterances of 100 to 300 frames x 1024 channels: 151 us with three, 132 with four); four channels a lane in float32 do not.
// PADDED: the wave has room for more states than there are.
template <typename T, int R, int S, bool GATE, int MODE, bool PADDED>
__global__ __launch_bounds__(64 * kScanWaves, R < 4 && R * S <= 8 ? 4 : 1) void scan_forward_kernel(ScanParams p) {
    constexpr int CH = 16 * R, NS = 4 * S, TILE = kScanTile;
    __shared__ __align__(16) float lds[kScanWaves][2 * TILE * (CH + NS)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* sD = lds[wave];
    float* sU = sD + TILE * CH;
    float* sB = sU + TILE * CH;
    float* sC = sB + TILE * NS;
    const int across = (p.blocks + kScanWaves - 1) / kScanWaves;
    const int groups = gridDim.x - (MODE == 0 ? p.clear : 0);
    if (MODE == 0 && (int)blockIdx.x >= groups) {
        clear_other_rows<T>(p.off, p.utts, p.frames, p.y, p.ld_y, p.channels, blockIdx.x - groups, p.clear);
        return;
    }
    for (int64_t task = blockIdx.x; task < p.units * across; task += groups) {
        const int64_t unit = task / across;
        const int block = (int)(task - unit * across) * kScanWaves + wave;
        ScanUnit u;
        if (block >= p.blocks || !scan_unit(p, unit, u)) continue;
        uniform_unit(u);
        const ScanLane<R, S, false> w(p, block);
        float A2[R][S], h[R][S], bias[R], skip[R], total[R];
        scan_load_A(p, w, A2);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            bias[r] = p.bias != nullptr && r < w.left ? p.bias[w.channel + r] : 0.0f;
            skip[r] = p.skip != nullptr && r < w.left ? p.skip[w.channel + r] : 0.0f;
            total[r] = 0.0f;
        }
        const int64_t place = unit * p.blocks + block;
        if (MODE == 0) {
            if (p.segment != 0) scan_load_lanes(p.seg_state, place, w, h);
            else scan_load_states(p.state_in, p, w, u.utt, h);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int s = 0; s < S; ++s) h[r][s] = 0.0f;
        }
        const int64_t frames = u.last - u.first;
        ScanTileReader<T, R, S, GATE, MODE == 0> reader(p, w, u.first);
        ScanTileRaw<T, R, S, GATE, MODE == 0> now, next;
        ScanRows<T> y(p.y, p.ld_y, u.first, w.row, w.channel);
        float* saved = nullptr;
        if (MODE == 0 && p.saved != nullptr)
            saved = p.saved + (scan_slot(u, u.first) * p.blocks + block) * (R * S * 64);
        if (frames > 0) reader.next(p, w, frames, now);
        for (int64_t done = 0; done < frames; done += TILE) {
            const int here = (int)min(frames - done, (int64_t)TILE);       // frames of this tile
            if (done + TILE < frames) reader.next(p, w, frames - done - TILE, next);
            Pack<float, R> step[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < R; ++r) step[i].v[r] = (float)now.dt[i].v[r] + bias[r];
            if (p.softplus)                              // (one branch, so that their latencies overlap)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < R; ++r) step[i].v[r] = softplus_f32(step[i].v[r]);
            wave_lds_fence();                            // the last tile has been read
            float odd = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                Pack<float, R> d = step[i], du;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    du.v[r] = d.v[r] * (float)now.x[i].v[r];
                    if (PADDED) odd = fmaf(du.v[r], 0.0f, odd);
                }
                if (here < TILE) {                       // a frame behind the last one changes nothing
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        d.v[r] = 4 * i + w.row < here ? d.v[r] : 0.0f;
                        du.v[r] = 4 * i + w.row < here ? du.v[r] : 0.0f;
                    }
                    arrive(d);                           // (a branch of the whole wave, not selections)
                }
                if (MODE == 1)
#pragma unroll
                    for (int r = 0; r < R; ++r) total[r] += d.v[r];
                store_pack(sD + (4 * i + w.row) * CH + w.col * R, d);
                store_pack(sU + (4 * i + w.row) * CH + w.col * R, du);
            }
            {
                Pack<float, S> b, c;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    b.v[s] = (float)now.b.v[s];
                    if (MODE == 0) c.v[s] = (float)now.c.v[s];
                }
                store_pack(sB + w.lane * S, b);
                if (MODE == 0) store_pack(sC + w.lane * S, c);
            }
            wave_lds_fence();
            Pack<T, R> out[4];
            const auto finish = [&](int i, int r, float v) {
                v = fmaf(skip[r], (float)now.x[i].v[r], v);
                if (GATE) {
                    const float z = (float)now.z[i].v[r];
                    v *= z * sigmoid_f32(z);
                }
                return (T)v;                             // the one rounding to the output's type
            };
            if (PADDED && __any(odd != 0.0f)) {
                // An infinite d x times the zeros of states that do not exist is not a number: such a tile goes frame by
                // frame, with a look at what exists (the loop below would take 3 to 9 % longer with one).
#pragma unroll 1
                for (int j = 0; j < TILE; ++j) {
                    if (saved != nullptr && j % kScanSaveEvery == 0 && j < here) {
                        scan_store_lanes(saved, 0, w, h);
                        saved += (int64_t)p.blocks * (R * S * 64);
                    }
                    ScanFrame<R, S> f;
                    f.template load<true, true>(w, j, sD, sU, nullptr, sB, sC);
                    Pack<float, R> sum;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        float v = 0.0f;
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            const float a = __builtin_amdgcn_exp2f(f.d.v[r] * A2[r][s]);
                            h[r][s] = w.exists(p, r, s) ? fmaf(a, h[r][s], f.du.v[r] * f.b.v[s]) : 0.0f;
                            v = fmaf(f.c.v[s], h[r][s], v);
                        }
                        v = halves_sum(v, v);
                        sum.v[r] = rows_sum(v, v);
                    }
                    store_pack(sU + j * CH + w.col * R, sum);            // (four lanes, the same values, over what is used)
                }
                wave_lds_fence();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const Pack<float, R> sum = load_pack<R>(sU + (4 * i + w.row) * CH + w.col * R);
#pragma unroll
                    for (int r = 0; r < R; ++r) out[i].v[r] = finish(i, r, sum.v[r]);
                }
            } else {
                ScanFrame<R, S> f;
                f.template load<true, MODE == 0>(w, 0, sD, sU, nullptr, sB, sC);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (MODE == 0 && i % 2 == 0 && saved != nullptr && 4 * i < here) {
                        scan_store_lanes(saved, 0, w, h);
                        saved += (int64_t)p.blocks * (R * S * 64);
                    }
                    float part[4][R];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        ScanFrame<R, S> ahead;               // the next frame's values are read while this one's are used
                        if (4 * i + j + 1 < TILE) ahead.template load<true, MODE == 0>(w, 4 * i + j + 1, sD, sU, nullptr, sB, sC);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            part[j][r] = 0.0f;
#pragma unroll
                            for (int s = 0; s < S; ++s) {
                                const float a = __builtin_amdgcn_exp2f(f.d.v[r] * A2[r][s]);
                                h[r][s] = fmaf(a, h[r][s], f.du.v[r] * f.b.v[s]);
                                if (MODE == 0) part[j][r] = fmaf(f.c.v[s], h[r][s], part[j][r]);
                            }
                        }
                        f = ahead;
                        __builtin_amdgcn_sched_barrier(0);   // (no more than that: registers)
                    }
                    if (MODE == 0) {
                        // the four rows' shares added up; row g is left with frame 4 i + g
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const float v = rows_sum(halves_sum(part[0][r], part[2][r]), halves_sum(part[1][r], part[3][r]));
                            out[i].v[r] = finish(i, r, v);
                        }
                        arrive(out[i]);                      // (computed here, and not in the branch that stores it)
                    }
                }
            }
            now = next;
            now.arrived();
            if (MODE == 0) {
                if (here == TILE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w.store(y, i, out[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * i + w.row < here) w.store(y, i, out[i]);
                }
                y.move(TILE);
            }
        }
        if (MODE == 0) {
            if (p.state_out != nullptr && u.tail) scan_store_states(p.state_out, p, w, u.utt, h);
        } else {
            scan_clear_absent(p, w, h);
            scan_store_lanes(p.seg_state, place, w, h);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float v = rows_sum(total[r], total[r]);
                total[r] = halves_sum(v, v);
            }
            if (w.row == 0) {
                Pack<float, R> v;
#pragma unroll
                for (int r = 0; r < R; ++r) v.v[r] = total[r];
                store_pack(p.seg_sum + place * CH + w.col * R, v);
            }
        }
    }
}

// The pieces of an utterance joined: seg_state holds what each piece's frames add to the state
// (REVERSE: to the gradient of the state before it), and is replaced by the state that enters the piece
// (the gradient that enters it from behind).  A workgroup has four values of each lane of one channel block;
// its waves take a run of pieces each, add them up from zero, hand the result to the waves behind them through LDS, and
// walk over their run again with the state that enters it.
// (Few pieces keep few waves busy: with seven of them a workgroup of 4 takes 4.7 us and one of 16 6.6, with 125 19.8 and
// 11.6.)
// A state that is zero stays zero, and an infinite one infinite, as they do over the piece's frames one after the other:
// the growth over all of a piece (an A above zero, or steps below) may be beyond 32 bits while that of every frame is not,
// and its decay may be 0.
__device__ __forceinline__ float scan_join(float decay, float h, float own) {
    const bool scaled = h != 0.0f && fabsf(h) < __builtin_huge_valf();
    return fmaf(scaled ? decay : 1.0f, h, own);
}
constexpr int kJoinWaves = 16;
inline int scan_join_threads(const ScanParams& p) { return 64 * (p.frames / (p.segment * p.utts) < 16 ? 4 : kJoinWaves); }
template <int R, int S, bool REVERSE>
__global__ __launch_bounds__(64 * kJoinWaves) void scan_join_kernel(ScanParams p) {
    constexpr int CH = 16 * R, QUADS = R * S / 4, AHEAD = 4;
    __shared__ float lds[kJoinWaves][2][64][4];
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    for (int64_t task = blockIdx.x; task < p.utts * p.blocks * QUADS; task += gridDim.x) {
        const int q = (int)(task % QUADS);
        const int64_t rest = task / QUADS, utt = rest / p.blocks;
        const int block = (int)(rest - utt * p.blocks);
        const ScanLane<R, S, false> w(p, block);
        float A2[4], h[4], decay[4];
        const float* enter = REVERSE ? p.dstate_out : p.state_in;
        float from[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = (q * 4 + k) / S, s = w.state + (q * 4 + k) % S;
            const bool in = r < w.left && s < p.states;
            A2[k] = in ? scan_log2_decay(p.A[(int64_t)(w.channel + r) * p.states + s]) : 0.0f;
            from[k] = in && enter != nullptr ? enter[(utt * p.channels + w.channel + r) * p.states + s] : 0.0f;
            h[k] = decay[k] = 0.0f;
        }
        int64_t begin, end;
        scan_bounds(p, utt, begin, end);
        const int64_t base = begin / p.segment + utt;
        const int64_t pieces = max((end - begin + p.segment - 1) / p.segment, (int64_t)1);
        const int64_t run = (pieces + waves - 1) / waves;
        const int64_t k0 = min(wave * run, pieces), k1 = min(k0 + run, pieces);
        auto place = [&](int64_t k) { return (base + (REVERSE ? pieces - 1 - k : k)) * p.blocks + block; };
        auto walk = [&](bool write) {
            for (int64_t k = k0; k < k1; k += AHEAD) {
                Pack<float, 4> own[AHEAD];
                float sum[AHEAD][4];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    const int64_t at = place(min(k + a, k1 - 1));
                    own[a] = load_pack<4>(p.seg_state + ((at * QUADS + q) * 64 + w.lane) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[a][e] = p.seg_sum[at * CH + w.col * R + (q * 4 + e) / S];
                }
                float by[AHEAD][4];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) by[a][e] = __builtin_amdgcn_exp2f(sum[a][e] * A2[e]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    if (k + a >= k1) break;
                    if (write) {
                        Pack<float, 4> v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v.v[e] = h[e];
                        store_pack(p.seg_state + ((place(k + a) * QUADS + q) * 64 + w.lane) * 4, v);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[e] = scan_join(by[a][e], h[e], own[a].v[e]);
                        decay[e] += sum[a][e];
                    }
                }
            }
        };
        walk(false);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lds[wave][0][w.lane][e] = h[e];
            lds[wave][1][w.lane][e] = decay[e];
            h[e] = from[e];
        }
        __syncthreads();
        for (int before = 0; before < wave; ++before)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                h[e] = scan_join(__builtin_amdgcn_exp2f(lds[before][1][w.lane][e] * A2[e]), h[e], lds[before][0][w.lane][e]);
        walk(true);
        __syncthreads();                                 // (the next task's results go to the same place)
    }
}

// ---- backward -----------------------------------------------------------------------------
//
// Backwards in time, g_{t-1} = exp(d_t A) (dp_t C_t + g_t) is what the loss owes to the state before
// frame t.  The states themselves are saved by the forward pass before every eighth frame and computed
// again from there, in registers.  Sums over the states (dd, dx, the gated sum) cross the four lanes that share
// channels, here neighbours (two quad permutations per sum); sums over the channels (dB, dC) cross the 16 lanes that
// share states: the first two of their four steps exchange whole halves and rows between two
// registers, so that each step halves the number of registers too.
//
// What does not exist (channels and states of a block, frames behind the last) has zeros for all that is its own, which an
// infinite state or input of those that there are would turn into NaN; it is kept from that.  An infinite gradient is not kept
// from it, nor an infinite C: sums that the definition makes infinite may be NaN then, finite ones stay.

template <typename T, int R, int S, bool GATE>
struct ScanOctetRaw {
    Pack<T, R> x[2], dt[2], z[2], dy[2];
    Pack<T, S> b, c;             // (lanes 32 .. 63 the same as lanes 0 .. 31)
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            arrive(x[i]);
            arrive(dt[i]);
            if (GATE) arrive(z[i]);
            arrive(dy[i]);
        }
        arrive(b);
        arrive(c);
    }
};
template <typename T, int R, int S, bool GATE>
struct ScanOctetReader {
    ScanRows<T> x, dt, z, dy, b, c;
    bool all_states;
    // `first`: the first frame of the octet that is read first; later ones lie before it
    __device__ __forceinline__ ScanOctetReader(const ScanParams& p, const ScanLane<R, S, true>& w, int64_t first) {
        const int s0 = w.group * p.states + (w.lane & 3) * S, t = (w.lane & 31) >> 2;
        x = ScanRows<T>(p.x, p.ld_x, first, w.row, w.channel);
        dt = ScanRows<T>(p.dt, p.ld_dt, first, w.row, w.channel);
        if (GATE) z = ScanRows<T>(p.gate, p.ld_gate, first, w.row, w.channel);
        dy = ScanRows<T>(p.dy, p.ld_dy, first, w.row, w.channel);
        b = ScanRows<T>(p.B, p.ld_B, first, t, s0);
        c = ScanRows<T>(p.C, p.ld_C, first, t, s0);
        all_states = p.states == 4 * S;
    }
    __device__ __forceinline__ void next(const ScanParams& p, const ScanLane<R, S, true>& w, int frames,
                                         ScanOctetRaw<T, R, S, GATE>& to) {
        const int last = frames - 1;
        if (last == kScanSaveEvery - 1 && w.full) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                to.x[i] = x.template load<R>(4 * i);
                to.dt[i] = dt.template load<R>(4 * i);
                if (GATE) to.z[i] = z.template load<R>(4 * i);
                to.dy[i] = dy.template load<R>(4 * i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                to.x[i] = w.load_any(x, i, last);
                to.dt[i] = w.load_any(dt, i, last);
                if (GATE) to.z[i] = w.load_any(z, i, last);
                to.dy[i] = w.load_any(dy, i, last);
            }
        }
        if (last == kScanSaveEvery - 1 && all_states) {
            to.b = b.template load<S>(0);
            to.c = c.template load<S>(0);
        } else {
            const int s0 = (w.lane & 3) * S, t = (w.lane & 31) >> 2;
            to.b = scan_load_bc<S>(b, t, last, w.group, s0, p.states);
            to.c = scan_load_bc<S>(c, t, last, w.group, s0, p.states);
        }
        x.move(-kScanSaveEvery);
        dt.move(-kScanSaveEvery);
        if (GATE) z.move(-kScanSaveEvery);
        dy.move(-kScanSaveEvery);
        b.move(-kScanSaveEvery);
        c.move(-kScanSaveEvery);
    }
};

// Sums over the 16 lanes that share states: lane 4 col + row gets of (lanes 0 .. 31: b, lanes 32 .. 63: c) the values
// odd S / 2 .. (odd rows of 16 lanes the second half of them; S = 1: all rows the one).
template <int S>
__device__ __forceinline__ void scan_sum_channels(const float (&b)[S], const float (&c)[S], float (&out)[S > 1 ? S / 2 : 1]) {
    float half[S];
#pragma unroll
    for (int s = 0; s < S; ++s) half[s] = halves_sum(b[s], c[s]);
#pragma unroll
    for (int s = 0; s < (S > 1 ? S / 2 : 1); ++s) {
        float v = rows_sum(half[s], half[S > 1 ? s + S / 2 : 0]);
        v += dpp_mov<0x124>(v);     // row_ror:4
        v += dpp_mov<0x128>(v);     // row_ror:8
        out[s] = v;
    }
}

// MODE 0: the gradients.  MODE 1: only what a piece adds to the gradient of the state before it,
// and the sum of its steps.  The states and decays of eight frames are held at once; with 64 states these are more
// registers than two waves per SIMD have, and one wave with all of them takes half the time of two that spill (64
// utterances of 100 to 300 frames x 1536 channels, forward and backward: 3.44 ms, now 1.69).
// PART: there are blocks with channels or states that do not exist (a branch over them costs whole blocks 1 %).
template <typename T, int R, int S, bool GATE, int MODE, bool PART>
__global__ __launch_bounds__(64 * kScanWaves, R * S > 8 ? 1 : 2) void scan_backward_kernel(ScanParams p) {
    constexpr int CH = 16 * R, NS = 4 * S, TILE = kScanSaveEvery;
    constexpr float kLn2 = 0.693147180559945309f;
    constexpr int kKept = GATE ? 6 : 4;  // 2 (x, slope of the step, gradient by the gate over the ungated output)
    __shared__ __align__(16) float lds[kScanWaves][TILE * (5 * CH + 4 * NS) + (MODE == 0 ? 64 * (R * S + 2 * R + kKept * R) : 0)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* sD = lds[wave];               // steps
    float* sU = sD + TILE * CH;          // step times x
    float* sP = sU + TILE * CH;          // gradient of the ungated output
    float* oU = sU;                      // sums over the states: dh B (in the place of what the frame has used)
    float* oD = sP + TILE * CH;          // dh a h A
    float* oY = oD + TILE * CH;          // C h
    float* sB = oY + TILE * CH;
    float* sC = sB + TILE * NS;
    float* oBC = sC + TILE * NS;         // [frame][B, C][state]: sums over the channels
    float* acc = oBC + 2 * TILE * NS;    // [R S + 2 R][64]: dA, dskip, dbias of the frames so far
    // what both ends of an octet's work need of a lane's own frames lies in LDS in between
    float* kept = acc + 64 * (R * S + 2 * R) + (threadIdx.x & 63) * R;
    const int across = (p.blocks + kScanWaves - 1) / kScanWaves;
    for (int64_t task = blockIdx.x; task < p.parts * across; task += gridDim.x) {
        const int64_t part = task / across;
        const int block = (int)(task - part * across) * kScanWaves + wave;
        if (block >= p.blocks) continue;
        const ScanLane<R, S, true> w(p, block);
        float A2[R][S], bias[R], skip[R], dA[R][S], dskip[R], dbias[R], total[R];
        scan_load_A(p, w, A2);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            bias[r] = p.bias != nullptr && r < w.left ? p.bias[w.channel + r] : 0.0f;
            skip[r] = p.skip != nullptr && r < w.left ? p.skip[w.channel + r] : 0.0f;
            dskip[r] = dbias[r] = 0.0f;
#pragma unroll
            for (int s = 0; s < S; ++s) dA[r][s] = 0.0f;
        }
        if (MODE == 0)
#pragma unroll
            for (int k = 0; k < R * S + 2 * R; ++k) acc[k * 64 + w.lane] = 0.0f;
        // frames summed in registers go to LDS every 256 frames: a long sum's error grows with the
        // root of its length, and two short ones after another keep it near that of the shorter
        int held = 0;
        auto flush = [&]() {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    acc[(r * S + s) * 64 + w.lane] += dA[r][s];
                    dA[r][s] = 0.0f;
                }
                acc[(R * S + r) * 64 + w.lane] += dskip[r];
                acc[(R * S + R + r) * 64 + w.lane] += dbias[r];
                dskip[r] = dbias[r] = 0.0f;
            }
            held = 0;
        };
        for (int64_t unit = part; unit < p.units; unit += p.parts) {
            ScanUnit u;
            if (!scan_unit(p, unit, u)) continue;
            uniform_unit(u);
            const int64_t place = unit * p.blocks + block;
            float g[R][S];
            if (MODE == 0) {
                if (p.segment != 0) scan_load_lanes(p.seg_state, place, w, g);
                else scan_load_states(p.dstate_out, p, w, u.utt, g);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    total[r] = 0.0f;
#pragma unroll
                    for (int s = 0; s < S; ++s) g[r][s] = 0.0f;
                }
            }
            const int64_t octets = (u.last - u.first + TILE - 1) / TILE;
            const int64_t begin = u.first + (octets - 1) * TILE;           // of the last octet
            ScanOctetReader<T, R, S, GATE> reader(p, w, begin);
            ScanOctetRaw<T, R, S, GATE> now, next;
            ScanRows<T> dx, ddt, dz;
            if (MODE == 0) {
                dx = ScanRows<T>(p.dx, p.ld_dx, begin, w.row, w.channel);
                ddt = ScanRows<T>(p.ddt, p.ld_ddt, begin, w.row, w.channel);
                if (GATE) dz = ScanRows<T>(p.dgate, p.ld_dgate, begin, w.row, w.channel);
            }
            const float* saved = MODE == 0 ? p.saved + (scan_slot(u, begin) * p.blocks + block) * (R * S * 64) : nullptr;
            float h0[R][S];
            int frames = (int)(u.last - begin);
            if (octets > 0) {
                reader.next(p, w, frames, now);
                if (MODE == 0) scan_load_lanes(saved, 0, w, h0);
            }
#pragma unroll 1
            for (int64_t o = octets - 1; o >= 0; --o) {
                const int64_t t0 = u.first + o * TILE;
                float h0next[R][S];
                if (MODE == 1 && o > 0) reader.next(p, w, TILE, next);
                Pack<float, R> step[2], slope[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        step[i].v[r] = (float)now.dt[i].v[r] + bias[r];
                        slope[i].v[r] = 1.0f;
                    }
                if (p.softplus)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            float by;
                            step[i].v[r] = softplus_f32(step[i].v[r], by);
                            slope[i].v[r] = by;
                        }
                wave_lds_fence();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    Pack<float, R> d = step[i], du, q, x, by_gate;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        x.v[r] = (float)now.x[i].v[r];
                        du.v[r] = d.v[r] * x.v[r];
                        q.v[r] = (float)now.dy[i].v[r];
                        if (GATE) {
                            const float z = (float)now.z[i].v[r], sig = sigmoid_f32(z), by = q.v[r] * sig;
                            q.v[r] = by * z;
                            by_gate.v[r] = fmaf(q.v[r], 1.0f - sig, by);
                        }
                    }
                    if (MODE == 0) {
                        store_pack(kept + i * 64 * R, x);
                        store_pack(kept + (2 + i) * 64 * R, slope[i]);
                        if (GATE) store_pack(kept + (4 + i) * 64 * R, by_gate);
                    }
                    if (frames < TILE || !w.full) {      // what does not exist adds nothing to anything
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const bool in = 4 * i + w.row < frames && r < w.left;
                            d.v[r] = in ? d.v[r] : 0.0f;
                            du.v[r] = in ? du.v[r] : 0.0f;
                            q.v[r] = in ? q.v[r] : 0.0f;
                        }
                    }
                    if (MODE == 1)
#pragma unroll
                        for (int r = 0; r < R; ++r) total[r] += d.v[r];
                    store_pack(sD + (4 * i + w.row) * CH + w.col * R, d);
                    store_pack(sU + (4 * i + w.row) * CH + w.col * R, du);
                    store_pack(sP + (4 * i + w.row) * CH + w.col * R, q);
                }
                {
                    Pack<float, S> b, c;
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        b.v[s] = (float)now.b.v[s];
                        c.v[s] = (float)now.c.v[s];
                    }
                    store_pack(sB + (w.lane & 31) * S, b);
                    store_pack(sC + (w.lane & 31) * S, c);
                }
                wave_lds_fence();
                if (MODE == 1) {
#pragma unroll
                    for (int j = TILE - 1; j >= 0; --j) {
                        ScanFrame<R, S> f;
                        f.template load<false, true>(w, j, sD, nullptr, sP, sB, sC);
#pragma unroll
                        for (int r = 0; r < R; ++r)
#pragma unroll
                            for (int s = 0; s < S; ++s)
                                g[r][s] = fmaf(f.q.v[r], f.c.v[s], g[r][s]) * __builtin_amdgcn_exp2f(f.d.v[r] * A2[r][s]);
                    }
                    now = next;
                    now.arrived();
                    frames = TILE;
                    continue;
                }
                float* to_bc = oBC + (w.lane >> 5) * NS + w.state + (S > 1 ? ((w.lane >> 4) & 1) * (S / 2) : 0);
                float a[TILE][R][S], h[TILE + 1][R][S];
                constexpr bool kAhead = R * S <= 4;
                ScanFrame<R, S> ahead;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int s = 0; s < S; ++s) h[0][r][s] = h0[r][s];
#pragma unroll
                for (int k = 0; k < TILE; ++k) {
                    ScanFrame<R, S> f;
                    if (!kAhead || k == 0) f.template load<true, false>(w, k, sD, sU, nullptr, sB, sC);
                    else f = ahead;
                    if (kAhead && k + 1 < TILE) ahead.template load<true, false>(w, k + 1, sD, sU, nullptr, sB, sC);
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            a[k][r][s] = __builtin_amdgcn_exp2f(f.d.v[r] * A2[r][s]);
                            h[k + 1][r][s] = fmaf(a[k][r][s], h[k][r][s], f.du.v[r] * f.b.v[s]);
                        }
                    if (k % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                }
                if (PART && (!w.full || p.states != NS)) {
                    // Channels and states that do not exist have the last channel's values, or zeros, and their states are
                    // no one's concern until an infinity makes them NaN, which the sums below would take up.
                    float odd = 0.0f;
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int s = 0; s < S; ++s) odd = fmaf(h[TILE][r][s], 0.0f, odd);
                    if (__any(odd != 0.0f)) {
#pragma unroll
                        for (int k = 0; k <= TILE; ++k)
#pragma unroll
                            for (int r = 0; r < R; ++r)
#pragma unroll
                                for (int s = 0; s < S; ++s) {
                                    h[k][r][s] = w.exists(p, r, s) ? h[k][r][s] : 0.0f;
                                    if (k < TILE) a[k][r][s] = w.exists(p, r, s) ? a[k][r][s] : 0.0f;
                                }
                    }
                }
#pragma unroll
                for (int k = TILE - 1; k >= 0; --k) {
                    // A frame behind the utterance's last adds nothing to dA, but its zeros would, times an infinite
                    // state.  It is passed by, or left out of that sum alone where the next frame's values are read ahead
                    // (64 utterances of 100 to 300 frames x 1024 channels, forward and backward, 7 states: 255 us and 249;
                    // 16 states in float32 with a gate 304 and 321).
                    const bool live = k == 0 || k < frames;
                    ScanFrame<R, S> f;
                    if (kAhead) {
                        if (k == TILE - 1) f.template load<true, true>(w, k, sD, sU, sP, sB, sC);
                        else f = ahead;
                        if (k > 0) ahead.template load<true, true>(w, k - 1, sD, sU, sP, sB, sC);
                    }
                    if (kAhead || live) {
                        if (!kAhead) f.template load<true, true>(w, k, sD, sU, sP, sB, sC);
                        float db[S], dc[S];
                        Pack<float, R> su, sd, sy;
#pragma unroll
                        for (int s = 0; s < S; ++s) db[s] = dc[s] = 0.0f;
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            float vu = 0.0f, vd = 0.0f, vy = 0.0f;
#pragma unroll
                            for (int s = 0; s < S; ++s) {
                                const float dh = fmaf(f.q.v[r], f.c.v[s], g[r][s]);
                                dc[s] = fmaf(f.q.v[r], h[k + 1][r][s], dc[s]);
                                if (GATE) vy = fmaf(f.c.v[s], h[k + 1][r][s], vy);
                                db[s] = fmaf(dh, f.du.v[r], db[s]);
                                vu = fmaf(dh, f.b.v[s], vu);
                                g[r][s] = dh * a[k][r][s];
                                const float m = g[r][s] * h[k][r][s];
                                vd = fmaf(m, A2[r][s], vd);
                                dA[r][s] = !kAhead || live ? fmaf(m, f.d.v[r], dA[r][s]) : dA[r][s];
                            }
                            su.v[r] = quad_sum(vu);
                            sd.v[r] = quad_sum(vd);
                            if (GATE) sy.v[r] = quad_sum(vy);
                        }
                        store_pack(oU + k * CH + w.col * R, su);        // (four lanes, the same values)
                        store_pack(oD + k * CH + w.col * R, sd);
                        if (GATE) store_pack(oY + k * CH + w.col * R, sy);
                        constexpr int HALF = S > 1 ? S / 2 : 1;
                        float sums[HALF];
                        scan_sum_channels<S>(db, dc, sums);
                        Pack<float, HALF> v;
#pragma unroll
                        for (int s = 0; s < HALF; ++s) v.v[s] = sums[s];
                        store_pack(to_bc + k * 2 * NS, v);              // (the lanes of a row, the same values)
                    }
                    // What the next octet needs is asked for when the last frame's registers are free.
                    if (k == TILE - 1 && o > 0) {
                        saved -= (int64_t)p.blocks * (R * S * 64);
                        scan_load_lanes(saved, 0, w, h0next);
                    }
                    if (k == TILE - 2 && o > 0) reader.next(p, w, TILE, next);
                    __builtin_amdgcn_sched_barrier(0);
                }
                wave_lds_fence();
                const Pack<float, S> sums = load_pack<S>(oBC + w.lane * S);
                Pack<T, R> vx[2], vt[2], vz[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bool live = 4 * i + w.row < frames;
                    const Pack<float, R> vu = load_pack<R>(oU + (4 * i + w.row) * CH + w.col * R);
                    const Pack<float, R> vd = load_pack<R>(oD + (4 * i + w.row) * CH + w.col * R);
                    Pack<float, R> vy;
                    if (GATE) vy = load_pack<R>(oY + (4 * i + w.row) * CH + w.col * R);
                    const Pack<float, R> d = load_pack<R>(sD + (4 * i + w.row) * CH + w.col * R);
                    const Pack<float, R> dp = load_pack<R>(sP + (4 * i + w.row) * CH + w.col * R);
                    const Pack<float, R> own = load_pack<R>(kept + i * 64 * R), by_step = load_pack<R>(kept + (2 + i) * 64 * R);
                    Pack<float, R> by_gate;
                    if (GATE) by_gate = load_pack<R>(kept + (4 + i) * 64 * R);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float x = own.v[r];
                        vx[i].v[r] = (T)fmaf(vu.v[r], d.v[r], dp.v[r] * skip[r]);
                        float v = fmaf(vd.v[r], kLn2, vu.v[r] * x) * by_step.v[r];
                        vt[i].v[r] = (T)v;
                        if (frames < TILE) v = live ? v : 0.0f;
                        dbias[r] += v;
                        dskip[r] = fmaf(dp.v[r], frames < TILE ? (live ? x : 0.0f) : x, dskip[r]);
                        if (GATE) vz[i].v[r] = (T)(by_gate.v[r] * fmaf(skip[r], x, vy.v[r]));
                    }
                }
                held += TILE;
                if (held >= 256) flush();
                now = next;
                now.arrived();
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        h0[r][s] = h0next[r][s];
                        arrive(h0[r][s]);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (4 * i + w.row < frames) {
                        w.store(dx, i, vx[i]);
                        w.store(ddt, i, vt[i]);
                        if (GATE) w.store(dz, i, vz[i]);
                    }
                }
                dx.move(-TILE);
                ddt.move(-TILE);
                if (GATE) dz.move(-TILE);
                if ((w.lane >> 3) < frames)
                    store_global<S, float>((GlobalChar*)(p.part_bc + ((int64_t)block * p.frames + t0) * 2 * NS), w.lane * S * 4, sums);
                frames = TILE;
            }
            if (MODE == 0) {
                if (p.dstate_in != nullptr && u.head) scan_store_states(p.dstate_in, p, w, u.utt, g);
            } else {
                scan_clear_absent(p, w, g);
                scan_store_lanes(p.seg_state, place, w, g);
                Pack<float, R> v;
#pragma unroll
                for (int r = 0; r < R; ++r) v.v[r] = quad_sum(total[r]);
                if (w.row == 0) store_pack(p.seg_sum + place * CH + w.col * R, v);
            }
        }
        if (MODE == 0) {
            flush();
            const int64_t place = part * p.blocks + block;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float vs = quad_sum(acc[(R * S + r) * 64 + w.lane]);
                const float vb = quad_sum(acc[(R * S + R + r) * 64 + w.lane]);
                if (w.row == 0) {
                    p.part_vec[(place * 2 + 0) * CH + w.col * R + r] = vs;
                    p.part_vec[(place * 2 + 1) * CH + w.col * R + r] = vb;
                }
#pragma unroll
                for (int s = 0; s < S; ++s) dA[r][s] = acc[(r * S + s) * 64 + w.lane];
            }
            scan_store_lanes(p.part_A, place, w, dA);
        }
    }
}

// dA, dskip, dbias: the parts of a channel block added up, always in the same order.  Workgroup (block, k):
// k < R S / 4: quads k of dA; k == R S / 4: the two vectors.  Wave w takes every fourth part.
template <int R, int S>
__device__ __forceinline__ void scan_sum_parts(const ScanParams& p, int task) {
    constexpr int CH = 16 * R, QUADS = R * S / 4;
    __shared__ double sum[4][64][4];
    const int block = task / (QUADS + 1), k = task % (QUADS + 1);
    const int wave = threadIdx.x >> 6;
    const ScanLane<R, S, false> w(p, block);
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t part = wave; part < p.parts; part += 4) {
        const int64_t place = part * p.blocks + block;
        if (k < QUADS) {
            const Pack<float, 4> q = load_pack<4>(p.part_A + ((place * QUADS + k) * 64 + w.lane) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += (double)q.v[i];
        } else if (w.lane < CH) {
            v[0] += (double)p.part_vec[(place * 2 + 0) * CH + w.lane];
            v[1] += (double)p.part_vec[(place * 2 + 1) * CH + w.lane];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[wave][w.lane][i] = v[i];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (sum[0][w.lane][i] + sum[1][w.lane][i]) + (sum[2][w.lane][i] + sum[3][w.lane][i]);
    if (k < QUADS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (k * 4 + i) / S, s = w.state + (k * 4 + i) % S;
            if (r < w.left && s < p.states) p.dA[(int64_t)(w.channel + r) * p.states + s] = (float)v[i];
        }
    } else if (w.lane < CH) {
        const int base = (block % p.group_blocks) * CH + w.lane;
        if (base < p.per_group) {
            const int c = (block / p.group_blocks) * p.per_group + base;
            if (p.dskip != nullptr) p.dskip[c] = (float)v[0];
            if (p.dbias != nullptr) p.dbias[c] = (float)v[1];
        }
    }
}

// dB, dC: the channel blocks of a group added up.  One thread per frame, group, B or C, and state.
template <typename T, int S>
__device__ __forceinline__ void scan_sum_bc(const ScanParams& p, int64_t group, int64_t groups) {
    constexpr int NS = 4 * S;
    const int64_t first = min(max(p.off[0], (int64_t)0), p.frames);
    const int64_t last = min(max(p.off[p.utts], first), p.frames);
    const int64_t total = (last - first) * p.groups * 2 * NS;
    for (int64_t i = group * 256 + threadIdx.x; i < total; i += groups * 256) {
        const int e = (int)(i % (2 * NS)), state = e % NS;
        const int64_t rest = i / (2 * NS);
        const int g = (int)(rest % p.groups);
        const int64_t t = first + rest / p.groups;
        const float* from = p.part_bc + ((int64_t)g * p.group_blocks * p.frames + t) * 2 * NS + e;
        const int64_t pitch = p.frames * 2 * NS;
        float v = 0.0f;
        int k = 0;
        for (; k + 8 <= p.group_blocks; k += 8, from += 8 * pitch) {         // eight loads in flight
            float q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = from[j * pitch];
            v += ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
        }
        for (; k < p.group_blocks; ++k, from += pitch) v += from[0];
        if (state < p.states) {
            const int64_t at = (int64_t)g * p.states + state;
            if (e < NS) ((T*)p.dB)[t * p.ld_dB + at] = (T)v;
            else ((T*)p.dC)[t * p.ld_dC + at] = (T)v;
        }
    }
}

// All in one launch: the first workgroups take the parameters' parts, the last ones the gradients of the frames that belong
// to no utterance, which are zero, the others dB and dC.
template <typename T, int R, int S>
__global__ __launch_bounds__(256) void scan_sum_kernel(ScanParams p) {
    const unsigned parts = (unsigned)p.blocks * (R * S / 4 + 1), clear = gridDim.x - p.clear;
    if (blockIdx.x < parts) {
        scan_sum_parts<R, S>(p, (int)blockIdx.x);
    } else if (blockIdx.x < clear) {
        scan_sum_bc<T, S>(p, blockIdx.x - parts, clear - parts);
    } else {
        void* const to[5] = {p.dx, p.ddt, p.dgate, p.dB, p.dC};
        const int64_t ld[5] = {p.ld_dx, p.ld_ddt, p.ld_dgate, p.ld_dB, p.ld_dC};
#pragma unroll
        for (int k = 0; k < 5; ++k)
            if (to[k] != nullptr)
                clear_other_rows<T>(p.off, p.utts, p.frames, to[k], ld[k], k < 3 ? p.channels : p.groups * p.states,
                                    blockIdx.x - clear, p.clear);
    }
}

// ---- one frame of every stream --------------------------------------------------------------
// Four neighbouring lanes share a channel, four states (16 bytes) of it each at a time: a wave reads
// and writes whole lines of the states.  Bound by the launch for few streams, by the states'
// bytes (8 per channel and state) for many.
template <typename T>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanParams p, float* state, int64_t streams) {
    const int sub = threadIdx.x & 3;
    const int across = (p.channels + 63) / 64;
    for (int64_t task = blockIdx.x; task < streams * across; task += gridDim.x) {
        const int64_t row = task / across;
        const int c = (int)(task - row * across) * 64 + (int)(threadIdx.x >> 2);
        if (c >= p.channels) continue;                  // (four lanes at a time)
        const float x = (float)((const T*)p.x)[row * p.ld_x + c];
        const float raw = (float)((const T*)p.dt)[row * p.ld_dt + c] + (p.bias != nullptr ? p.bias[c] : 0.0f);
        const float d = p.softplus ? softplus_f32(raw) : raw;
        const float du = d * x;
        const int64_t bc = (int64_t)(c / p.per_group) * p.states;
        float* h = state + (row * p.channels + c) * p.states;
        const float* A = p.A + (int64_t)c * p.states;
        float y = 0.0f;
        for (int n0 = sub * 4; n0 < p.states; n0 += 16) {
            const int left = p.states - n0;
            Pack<float, 4> v = load_some<4>(h + n0, left);
            const Pack<float, 4> a = load_some<4>(A + n0, left);
            const Pack<T, 4> b = load_some<4>((const T*)p.B + row * p.ld_B + bc + n0, left);
            const Pack<T, 4> q = load_some<4>((const T*)p.C + row * p.ld_C + bc + n0, left);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v.v[k] = fmaf(exp_f32(d * scan_finite(a.v[k])), v.v[k], du * (float)b.v[k]);
                if (k < left) y = fmaf((float)q.v[k], v.v[k], y);        // (an infinite d x times their zeros is not a number)
            }
            store_some(h + n0, v, left);
        }
        y = quad_sum(y);
        if (p.skip != nullptr) y = fmaf(p.skip[c], x, y);
        if (p.gate != nullptr) {
            const float z = (float)((const T*)p.gate)[row * p.ld_gate + c];
            y *= z * sigmoid_f32(z);
        }
        if (sub == 0) ((T*)p.y)[row * p.ld_y + c] = (T)y;
    }
}

// ---- launches -------------------------------------------------------------------------------

constexpr int64_t kScanMostWorkgroups = 1 << 22;      // loops take what a grid cannot

inline unsigned scan_grid(int64_t tasks) {
    return (unsigned)(tasks < 1 ? 1 : tasks < kScanMostWorkgroups ? tasks : kScanMostWorkgroups);
}

// Whether utterances are ever cut into pieces: two channels a lane with 16 states are for batches that fill the device.
constexpr bool scan_cuts(int R, int S) { return !(R == 2 && S == 4); }

template <typename T, int R, int S, bool GATE>
int scan_forward_launch(const ScanParams& p, hipStream_t st) {
    const int64_t across = (p.blocks + kScanWaves - 1) / kScanWaves;
    if constexpr (scan_cuts(R, S)) if (p.segment != 0) {
        scan_forward_kernel<T, R, S, GATE, 1, false><<<scan_grid(p.units * across), 64 * kScanWaves, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
        scan_join_kernel<R, S, false><<<scan_grid(p.utts * p.blocks * (R * S / 4)), scan_join_threads(p), 0, st>>>(p);
        SRX_HIP(hipGetLastError());
    }
    if (p.order != nullptr) {
        scan_order_kernel<<<1, kScanOrdered, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
    }
    const unsigned wide = scan_grid(p.units * across) + p.clear;
    if (p.states != 4 * S) scan_forward_kernel<T, R, S, GATE, 0, true><<<wide, 64 * kScanWaves, 0, st>>>(p);
    else scan_forward_kernel<T, R, S, GATE, 0, false><<<wide, 64 * kScanWaves, 0, st>>>(p);
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

template <typename T, int R, int S, bool GATE>
int scan_backward_launch(const ScanParams& q, hipStream_t st) {
    ScanParams p = q;
    const int64_t across = (p.blocks + kScanWaves - 1) / kScanWaves;
    if constexpr (scan_cuts(R, S)) if (p.segment != 0) {
        const int64_t parts = p.parts;
        p.parts = p.units;
        scan_backward_kernel<T, R, S, GATE, 1, true><<<scan_grid(p.units * across), 64 * kScanWaves, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
        scan_join_kernel<R, S, true><<<scan_grid(p.utts * p.blocks * (R * S / 4)), scan_join_threads(p), 0, st>>>(p);
        SRX_HIP(hipGetLastError());
        p.parts = parts;
    }
    const unsigned wide = scan_grid(p.parts * across);
    if (p.per_group % (16 * R) != 0 || p.states != 4 * S) scan_backward_kernel<T, R, S, GATE, 0, true><<<wide, 64 * kScanWaves, 0, st>>>(p);
    else scan_backward_kernel<T, R, S, GATE, 0, false><<<wide, 64 * kScanWaves, 0, st>>>(p);
    SRX_HIP(hipGetLastError());
    const int64_t sums = p.utts > 0 ? p.frames * p.groups * 8 * S : 0;
    const unsigned more = sums > 0 ? scan_grid((sums + 255) / 256) : 0;
    scan_sum_kernel<T, R, S><<<(unsigned)(p.blocks * (R * S / 4 + 1)) + more + p.clear, 256, 0, st>>>(p);
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

// The shapes of a wave that there are: 16 R channels, 4 S states (p.wide = R, see ssm_scan.hip).
template <typename T, bool GATE>
int scan_dispatch(const ScanParams& p, bool backward, hipStream_t st) {
#define SRX_SCAN_CASE(R, S)                                                                   \
    if (p.states <= 4 * S && p.wide == R)                                                     \
        return backward ? scan_backward_launch<T, R, S, GATE>(p, st) : scan_forward_launch<T, R, S, GATE>(p, st);
    SRX_SCAN_CASE(4, 1)
    SRX_SCAN_CASE(2, 2)
    SRX_SCAN_CASE(2, 4)
    SRX_SCAN_CASE(1, 4)
    SRX_SCAN_CASE(1, 8)
    SRX_SCAN_CASE(1, 16)
#undef SRX_SCAN_CASE
    srx_set_error("selective scan: no kernel for %d states, %d channels a lane", p.states, p.wide);
    return SRX_EUNSUPPORTED;
}

// Defined once per element type (ssm_scan_f32.hip, ssm_scan_bf16.hip, ssm_scan_f16.hip).
template <typename T>
int scan_run(const ScanParams& p, bool backward, hipStream_t st);
template <typename T>
int scan_step_run(const ScanParams& p, float* state, int64_t streams, hipStream_t st);

#define SRX_SCAN_INSTANTIATE(T)                                                               \
    template <>                                                                               \
    int scan_run<T>(const ScanParams& p, bool backward, hipStream_t st) {                     \
        return p.gate != nullptr ? scan_dispatch<T, true>(p, backward, st)                    \
                                 : scan_dispatch<T, false>(p, backward, st);                  \
    }                                                                                         \
    template <>                                                                               \
    int scan_step_run<T>(const ScanParams& p, float* state, int64_t streams, hipStream_t st) { \
        const int64_t tasks = streams * ((p.channels + 63) / 64);                             \
        scan_step_kernel<T><<<scan_grid(tasks), 256, 0, st>>>(p, state, streams);             \
        SRX_HIP(hipGetLastError());                                                           \
        return SRX_OK;                                                                        \
    }
