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
    // frames
    const int64_t* off;
    int64_t utts, frames;
    const void *x, *dt, *B, *C, *gate;
    int64_t ld_x, ld_dt, ld_B, ld_C, ld_gate;
    // units: utterances (segment == 0) or pieces of `segment` frames of them
    int64_t units, segment;
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
        scan_bounds(p, unit, begin, end);
        w = {unit, begin, begin, end, true, true};
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

// Channels of a wave's block, and where they are.
template <int R, int S>
struct ScanLane {
    static constexpr int kChannels = 16 * R, kStates = 4 * S;
    int lane, row, col;
    int group, channel, left;    // first channel of this lane, how many of its R exist
    int state;                   // first state of this lane
    __device__ __forceinline__ ScanLane(const ScanParams& p, int block) {
        lane = threadIdx.x & 63;
        row = lane >> 4;
        col = lane & 15;
        group = block / p.group_blocks;
        const int base = (block - group * p.group_blocks) * kChannels + col * R;
        channel = group * p.per_group + base;
        left = min(max(p.per_group - base, 0), R);
        state = row * S;
    }
};

template <int R, int S>
__device__ __forceinline__ void scan_load_states(const float* from, const ScanParams& p, const ScanLane<R, S>& w,
                                                 int64_t utt, float (&h)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s)
            h[r][s] = from != nullptr && r < w.left && w.state + s < p.states
                          ? from[(utt * p.channels + w.channel + r) * p.states + w.state + s] : 0.0f;
}
template <int R, int S>
__device__ __forceinline__ void scan_store_states(float* to, const ScanParams& p, const ScanLane<R, S>& w,
                                                  int64_t utt, const float (&h)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (r < w.left && w.state + s < p.states)
                to[(utt * p.channels + w.channel + r) * p.states + w.state + s] = h[r][s];
}
// The same in the lanes' own order (whole lines per instruction, padded channels and states included).
template <int R, int S>
__device__ __forceinline__ void scan_load_lanes(const float* from, int64_t at, int lane, float (&h)[R][S]) {
    const float* base = from + (at * (R * S / 4) * 64 + lane) * 4;
#pragma unroll
    for (int q = 0; q < R * S / 4; ++q) {
        const Pack<float, 4> v = load_pack<4>(base + q * 256);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[(q * 4 + k) / S][(q * 4 + k) % S] = v.v[k];
    }
}
template <int R, int S>
__device__ __forceinline__ void scan_store_lanes(float* to, int64_t at, int lane, const float (&h)[R][S]) {
    float* base = to + (at * (R * S / 4) * 64 + lane) * 4;
#pragma unroll
    for (int q = 0; q < R * S / 4; ++q) {
        Pack<float, 4> v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v.v[k] = h[(q * 4 + k) / S][(q * 4 + k) % S];
        store_pack(base + q * 256, v);
    }
}
__device__ __forceinline__ int64_t scan_slot(const ScanUnit& u, int64_t t) {
    return u.begin / kScanSaveEvery + u.utt + (t - u.begin) / kScanSaveEvery;
}

// A log2(e), so that the decay is one product and the hardware's 2^x.
template <int R, int S>
__device__ __forceinline__ void scan_load_A(const ScanParams& p, const ScanLane<R, S>& w, float (&A2)[R][S]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int s = 0; s < S; ++s)
            A2[r][s] = r < w.left && w.state + s < p.states
                           ? p.A[(int64_t)(w.channel + r) * p.states + w.state + s] * 1.44269504088896341f : 0.0f;
}

// ---- forward ------------------------------------------------------------------------------

// A tile of frames on its way from memory: row g of the wave has frames 4 i + g.
template <typename T, int R, int S, bool GATE, bool WITH_Y>
struct ScanTileRaw {
    Pack<T, R> x[4], dt[4], z[4];
    Pack<T, S> b, c;
    __device__ __forceinline__ void load(const ScanParams& p, const ScanLane<R, S>& w, int64_t t0, int64_t last) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t t = min(t0 + 4 * i + w.row, last - 1);      // behind the last frame: it again, unused
            x[i] = load_some<R>((const T*)p.x + t * p.ld_x + w.channel, w.left);
            dt[i] = load_some<R>((const T*)p.dt + t * p.ld_dt + w.channel, w.left);
            if (GATE && WITH_Y) z[i] = load_some<R>((const T*)p.gate + t * p.ld_gate + w.channel, w.left);
        }
        const int64_t t = min(t0 + (w.lane >> 2), last - 1);
        const int s0 = (w.lane & 3) * S;
        b = load_some<S>((const T*)p.B + t * p.ld_B + (int64_t)w.group * p.states + s0, p.states - s0);
        if (WITH_Y) c = load_some<S>((const T*)p.C + t * p.ld_C + (int64_t)w.group * p.states + s0, p.states - s0);
    }
};

// MODE 0: the outputs.  MODE 1: only the last state of a piece and the sum of its steps.
template <typename T, int R, int S, bool GATE, int MODE>
__global__ __launch_bounds__(64 * kScanWaves) void scan_forward_kernel(ScanParams p) {
    constexpr int CH = 16 * R, NS = 4 * S, TILE = kScanTile;
    __shared__ float lds[kScanWaves][2 * TILE * (CH + NS)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* sD = lds[wave];
    float* sU = sD + TILE * CH;
    float* sB = sU + TILE * CH;
    float* sC = sB + TILE * NS;
    const int across = (p.blocks + kScanWaves - 1) / kScanWaves;
    for (int64_t task = blockIdx.x; task < p.units * across; task += gridDim.x) {
        const int64_t unit = task / across;
        const int block = (int)(task - unit * across) * kScanWaves + wave;
        ScanUnit u;
        if (block >= p.blocks || !scan_unit(p, unit, u)) continue;
        const ScanLane<R, S> w(p, block);
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
            if (p.segment != 0) scan_load_lanes(p.seg_state, place, w.lane, h);
            else scan_load_states(p.state_in, p, w, u.utt, h);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int s = 0; s < S; ++s) h[r][s] = 0.0f;
        }
        ScanTileRaw<T, R, S, GATE, MODE == 0> now, next;
        if (u.first < u.last) now.load(p, w, u.first, u.last);
        for (int64_t t0 = u.first; t0 < u.last; t0 += TILE) {
            if (t0 + TILE < u.last) next.load(p, w, t0 + TILE, u.last);
            wave_lds_fence();                            // the last tile has been read
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool live = t0 + 4 * i + w.row < u.last;
                Pack<float, R> d, du;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float raw = (float)now.dt[i].v[r] + bias[r];
                    const float step = p.softplus ? softplus_f32(raw) : raw;
                    d.v[r] = live ? step : 0.0f;         // a frame behind the last one changes nothing
                    du.v[r] = live ? step * (float)now.x[i].v[r] : 0.0f;
                    if (MODE == 1) total[r] += d.v[r];
                }
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
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (MODE == 0 && i % 2 == 0 && p.saved != nullptr && t0 + 4 * i < u.last)
                    scan_store_lanes(p.saved, scan_slot(u, t0 + 4 * i) * p.blocks + block, w.lane, h);
                float y[4][R];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const Pack<float, R> d = load_pack<R>(sD + (4 * i + j) * CH + w.col * R);
                    const Pack<float, R> du = load_pack<R>(sU + (4 * i + j) * CH + w.col * R);
                    const Pack<float, S> b = load_pack<S>(sB + (4 * i + j) * NS + w.state);
                    Pack<float, S> c;
                    if (MODE == 0) c = load_pack<S>(sC + (4 * i + j) * NS + w.state);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        y[j][r] = 0.0f;
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            const float a = __builtin_amdgcn_exp2f(d.v[r] * A2[r][s]);
                            h[r][s] = fmaf(a, h[r][s], du.v[r] * b.v[s]);
                            if (MODE == 0) y[j][r] = fmaf(c.v[s], h[r][s], y[j][r]);
                        }
                    }
                }
                if (MODE == 0) {
                    // the four rows' shares added up; row g is left with frame 4 i + g
                    Pack<T, R> out;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        float v = rows_sum(halves_sum(y[0][r], y[2][r]), halves_sum(y[1][r], y[3][r]));
                        v = fmaf(skip[r], (float)now.x[i].v[r], v);
                        if (GATE) {
                            const float z = (float)now.z[i].v[r];
                            v *= z * sigmoid_f32(z);
                        }
                        out.v[r] = (T)v;                 // the one rounding to the output's type
                    }
                    const int64_t t = t0 + 4 * i + w.row;
                    if (t < u.last) store_some((T*)p.y + t * p.ld_y + w.channel, out, w.left);
                }
            }
            now = next;
        }
        if (MODE == 0) {
            if (p.state_out != nullptr && u.tail) scan_store_states(p.state_out, p, w, u.utt, h);
        } else {
            scan_store_lanes(p.seg_state, place, w.lane, h);
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
// (the gradient that enters it from behind).  One wave per utterance and channel block walks over the
// pieces; its loads do not depend on one another.
template <int R, int S, bool REVERSE>
__global__ __launch_bounds__(64) void scan_join_kernel(ScanParams p) {
    constexpr int CH = 16 * R;
    for (int64_t task = blockIdx.x; task < p.utts * p.blocks; task += gridDim.x) {
        const int64_t utt = task / p.blocks;
        const int block = (int)(task - utt * p.blocks);
        const ScanLane<R, S> w(p, block);
        float A2[R][S], h[R][S];
        scan_load_A(p, w, A2);
        scan_load_states(REVERSE ? p.dstate_out : p.state_in, p, w, utt, h);
        int64_t begin, end;
        scan_bounds(p, utt, begin, end);
        const int64_t base = begin / p.segment + utt;
        const int64_t pieces = max((end - begin + p.segment - 1) / p.segment, (int64_t)1);
        for (int64_t k = 0; k < pieces; ++k) {
            const int64_t place = (base + (REVERSE ? pieces - 1 - k : k)) * p.blocks + block;
            float own[R][S];
            scan_load_lanes(p.seg_state, place, w.lane, own);
            const Pack<float, R> sum = load_pack<R>(p.seg_sum + place * CH + w.col * R);
            scan_store_lanes(p.seg_state, place, w.lane, h);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int s = 0; s < S; ++s)
                    h[r][s] = fmaf(__builtin_amdgcn_exp2f(sum.v[r] * A2[r][s]), h[r][s], own[r][s]);
        }
    }
}

// ---- backward -----------------------------------------------------------------------------
//
// Backwards in time, g_{t-1} = exp(d_t A) (dp_t C_t + g_t) is what the loss owes to the state before
// frame t.  The states themselves are saved by the forward pass before every eighth frame and computed
// again from there, in registers, four frames at a time: the first four frames' states of an
// octet are run through once to reach the second four.  Sums over the states (dd, dx, the gated sum)
// cross the rows of a wave, sums over the channels (dB, dC) its columns.

template <typename T, int R, int S, bool GATE>
struct ScanOctetRaw {
    Pack<T, R> x[2], dt[2], z[2], dy[2];
    Pack<T, S> bc;               // lanes 0 .. 31: B, lanes 32 .. 63: C
    __device__ __forceinline__ void load(const ScanParams& p, const ScanLane<R, S>& w, int64_t t0, int64_t last) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t t = min(t0 + 4 * i + w.row, last - 1);
            x[i] = load_some<R>((const T*)p.x + t * p.ld_x + w.channel, w.left);
            dt[i] = load_some<R>((const T*)p.dt + t * p.ld_dt + w.channel, w.left);
            if (GATE) z[i] = load_some<R>((const T*)p.gate + t * p.ld_gate + w.channel, w.left);
            dy[i] = load_some<R>((const T*)p.dy + t * p.ld_dy + w.channel, w.left);
        }
        const int64_t t = min(t0 + ((w.lane & 31) >> 2), last - 1);
        const int s0 = (w.lane & 3) * S;
        const T* from = w.lane < 32 ? (const T*)p.B + t * p.ld_B : (const T*)p.C + t * p.ld_C;
        bc = load_some<S>(from + (int64_t)w.group * p.states + s0, p.states - s0);
    }
};

// The sum of v[r] over the four rows; row g gets that of r = g (R = 4), g / 2 (R = 2), 0 (R = 1).
template <int R>
__device__ __forceinline__ float scan_rows(const float (&v)[R]) {
    if constexpr (R == 4) {
        return rows_sum(halves_sum(v[0], v[2]), halves_sum(v[1], v[3]));
    } else if constexpr (R == 2) {
        const float a = halves_sum(v[0], v[1]);
        return rows_sum(a, a);
    } else {
        const float a = halves_sum(v[0], v[0]);
        return rows_sum(a, a);
    }
}

// MODE 0: the gradients.  MODE 1: only what a piece adds to the gradient of the state before it,
// and the sum of its steps.
template <typename T, int R, int S, bool GATE, int MODE>
__global__ __launch_bounds__(64 * kScanWaves, 2) void scan_backward_kernel(ScanParams p) {
    constexpr int CH = 16 * R, NS = 4 * S, TILE = kScanSaveEvery;
    constexpr float kLn2 = 0.693147180559945309f;
    __shared__ float lds[kScanWaves][TILE * (6 * CH + 2 * NS) + 64 * (R * S + 2 * R)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* sD = lds[wave];               // steps
    float* sU = sD + TILE * CH;          // step times x
    float* sP = sU + TILE * CH;          // gradient of the ungated output
    float* oU = sP + TILE * CH;          // sums over the states: dh B
    float* oD = oU + TILE * CH;          // dh a h A
    float* oY = oD + TILE * CH;          // C h
    float* sB = oY + TILE * CH;
    float* sC = sB + TILE * NS;
    float* acc = sC + TILE * NS;         // [R S + 2 R][64]: dA, dskip, dbias of the frames so far
    const int across = (p.blocks + kScanWaves - 1) / kScanWaves;
    for (int64_t task = blockIdx.x; task < p.parts * across; task += gridDim.x) {
        const int64_t part = task / across;
        const int block = (int)(task - part * across) * kScanWaves + wave;
        if (block >= p.blocks) continue;
        const ScanLane<R, S> w(p, block);
        const int owner = R == 4 ? w.row : R == 2 ? w.row >> 1 : 0;      // the channel whose sums this row gets
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
        const int64_t unit0 = part * p.units / p.parts, unit1 = (part + 1) * p.units / p.parts;
        for (int64_t unit = unit0; unit < unit1; ++unit) {
            ScanUnit u;
            if (!scan_unit(p, unit, u)) continue;
            const int64_t place = unit * p.blocks + block;
            float g[R][S];
            if (MODE == 0) {
                if (p.segment != 0) scan_load_lanes(p.seg_state, place, w.lane, g);
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
            for (int64_t o = octets - 1; o >= 0; --o) {
                const int64_t t0 = u.first + o * TILE;
                ScanOctetRaw<T, R, S, GATE> now;
                now.load(p, w, t0, u.last);
                float h0[R][S];
                if (MODE == 0) scan_load_lanes(p.saved, scan_slot(u, t0) * p.blocks + block, w.lane, h0);
                wave_lds_fence();
                float step[2][R], dp[2][R];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bool live = t0 + 4 * i + w.row < u.last;
                    Pack<float, R> d, du, q;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float raw = (float)now.dt[i].v[r] + bias[r];
                        const float v = p.softplus ? softplus_f32(raw) : raw;
                        d.v[r] = live ? v : 0.0f;
                        du.v[r] = live ? v * (float)now.x[i].v[r] : 0.0f;
                        float dv = (float)now.dy[i].v[r];
                        if (GATE) {
                            const float z = (float)now.z[i].v[r];
                            dv *= z * sigmoid_f32(z);
                        }
                        q.v[r] = live ? dv : 0.0f;
                        step[i][r] = d.v[r];
                        dp[i][r] = q.v[r];
                        if (MODE == 1) total[r] += d.v[r];
                    }
                    store_pack(sD + (4 * i + w.row) * CH + w.col * R, d);
                    store_pack(sU + (4 * i + w.row) * CH + w.col * R, du);
                    store_pack(sP + (4 * i + w.row) * CH + w.col * R, q);
                }
                {
                    Pack<float, S> v;
#pragma unroll
                    for (int s = 0; s < S; ++s) v.v[s] = (float)now.bc.v[s];
                    store_pack((w.lane < 32 ? sB : sC) + (w.lane & 31) * S, v);
                }
                wave_lds_fence();
                if (MODE == 1) {
#pragma unroll
                    for (int j = TILE - 1; j >= 0; --j) {
                        const Pack<float, R> d = load_pack<R>(sD + j * CH + w.col * R);
                        const Pack<float, R> q = load_pack<R>(sP + j * CH + w.col * R);
                        const Pack<float, S> c = load_pack<S>(sC + j * NS + w.state);
#pragma unroll
                        for (int r = 0; r < R; ++r)
#pragma unroll
                            for (int s = 0; s < S; ++s)
                                g[r][s] = fmaf(q.v[r], c.v[s], g[r][s]) * __builtin_amdgcn_exp2f(d.v[r] * A2[r][s]);
                    }
                    continue;
                }
                // states before the second four frames
                float h4[R][S];
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int s = 0; s < S; ++s) h4[r][s] = h0[r][s];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const Pack<float, R> d = load_pack<R>(sD + j * CH + w.col * R);
                    const Pack<float, R> du = load_pack<R>(sU + j * CH + w.col * R);
                    const Pack<float, S> b = load_pack<S>(sB + j * NS + w.state);
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int s = 0; s < S; ++s)
                            h4[r][s] = fmaf(__builtin_amdgcn_exp2f(d.v[r] * A2[r][s]), h4[r][s], du.v[r] * b.v[s]);
                }
#pragma unroll
                for (int half = 1; half >= 0; --half) {
                    float a[4][R][S], h[5][R][S];
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int s = 0; s < S; ++s) h[0][r][s] = half ? h4[r][s] : h0[r][s];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int j = 4 * half + k;
                        const Pack<float, R> d = load_pack<R>(sD + j * CH + w.col * R);
                        const Pack<float, R> du = load_pack<R>(sU + j * CH + w.col * R);
                        const Pack<float, S> b = load_pack<S>(sB + j * NS + w.state);
#pragma unroll
                        for (int r = 0; r < R; ++r)
#pragma unroll
                            for (int s = 0; s < S; ++s) {
                                a[k][r][s] = __builtin_amdgcn_exp2f(d.v[r] * A2[r][s]);
                                h[k + 1][r][s] = fmaf(a[k][r][s], h[k][r][s], du.v[r] * b.v[s]);
                            }
                    }
#pragma unroll
                    for (int k = 3; k >= 0; --k) {
                        const int j = 4 * half + k;
                        const Pack<float, R> d = load_pack<R>(sD + j * CH + w.col * R);
                        const Pack<float, R> du = load_pack<R>(sU + j * CH + w.col * R);
                        const Pack<float, R> q = load_pack<R>(sP + j * CH + w.col * R);
                        const Pack<float, S> b = load_pack<S>(sB + j * NS + w.state);
                        const Pack<float, S> c = load_pack<S>(sC + j * NS + w.state);
                        float su[R], sd[R], sy[R], db[S], dc[S];
#pragma unroll
                        for (int s = 0; s < S; ++s) db[s] = dc[s] = 0.0f;
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            su[r] = sd[r] = sy[r] = 0.0f;
#pragma unroll
                            for (int s = 0; s < S; ++s) {
                                const float dh = fmaf(q.v[r], c.v[s], g[r][s]);
                                dc[s] = fmaf(q.v[r], h[k + 1][r][s], dc[s]);
                                if (GATE) sy[r] = fmaf(c.v[s], h[k + 1][r][s], sy[r]);
                                db[s] = fmaf(dh, du.v[r], db[s]);
                                su[r] = fmaf(dh, b.v[s], su[r]);
                                g[r][s] = dh * a[k][r][s];
                                const float m = g[r][s] * h[k][r][s];
                                sd[r] = fmaf(m, A2[r][s], sd[r]);
                                dA[r][s] = fmaf(m, d.v[r], dA[r][s]);
                            }
                        }
                        const int at = j * CH + w.col * R + owner;
                        oU[at] = scan_rows<R>(su);
                        oD[at] = scan_rows<R>(sd);
                        if (GATE) oY[at] = scan_rows<R>(sy);
                        Pack<float, S> out;
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            const float vb = row16_sum(db[s]), vc = row16_sum(dc[s]);
                            out.v[s] = w.col == 0 ? vb : vc;
                        }
                        if (w.col < 2 && t0 + j < u.last)
                            store_pack(p.part_bc + (((int64_t)block * p.frames + t0 + j) * 2 + w.col) * NS + w.state, out);
                    }
                }
                wave_lds_fence();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int64_t t = t0 + 4 * i + w.row;
                    const bool live = t < u.last;
                    const Pack<float, R> vu = load_pack<R>(oU + (4 * i + w.row) * CH + w.col * R);
                    const Pack<float, R> vd = load_pack<R>(oD + (4 * i + w.row) * CH + w.col * R);
                    Pack<float, R> vy;
                    if (GATE) vy = load_pack<R>(oY + (4 * i + w.row) * CH + w.col * R);
                    Pack<T, R> dx, ddt, dz;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float x = (float)now.x[i].v[r];
                        dx.v[r] = (T)fmaf(vu.v[r], step[i][r], dp[i][r] * skip[r]);
                        float v = fmaf(vd.v[r], kLn2, vu.v[r] * x);
                        if (p.softplus) v *= sigmoid_f32((float)now.dt[i].v[r] + bias[r]);
                        ddt.v[r] = (T)v;
                        if (live) {
                            dbias[r] += v;
                            dskip[r] = fmaf(dp[i][r], x, dskip[r]);
                        }
                        if (GATE) {
                            const float z = (float)now.z[i].v[r], sig = sigmoid_f32(z);
                            const float out = fmaf(skip[r], x, vy.v[r]);
                            dz.v[r] = (T)((float)now.dy[i].v[r] * out * sig * fmaf(z, 1.0f - sig, 1.0f));
                        }
                    }
                    if (live) {
                        store_some((T*)p.dx + t * p.ld_dx + w.channel, dx, w.left);
                        store_some((T*)p.ddt + t * p.ld_ddt + w.channel, ddt, w.left);
                        if (GATE) store_some((T*)p.dgate + t * p.ld_dgate + w.channel, dz, w.left);
                    }
                }
                held += TILE;
                if (held >= 256) flush();
            }
            if (MODE == 0) {
                if (p.dstate_in != nullptr && u.head) scan_store_states(p.dstate_in, p, w, u.utt, g);
            } else {
                scan_store_lanes(p.seg_state, place, w.lane, g);
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
        if (MODE == 0) {
            flush();
            const int64_t place = part * p.blocks + block;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v = rows_sum(acc[(R * S + r) * 64 + w.lane], acc[(R * S + r) * 64 + w.lane]);
                const float vs = halves_sum(v, v);
                v = rows_sum(acc[(R * S + R + r) * 64 + w.lane], acc[(R * S + R + r) * 64 + w.lane]);
                const float vb = halves_sum(v, v);
                if (w.row == 0) {
                    p.part_vec[(place * 2 + 0) * CH + w.col * R + r] = vs;
                    p.part_vec[(place * 2 + 1) * CH + w.col * R + r] = vb;
                }
#pragma unroll
                for (int s = 0; s < S; ++s) dA[r][s] = acc[(r * S + s) * 64 + w.lane];
            }
            scan_store_lanes(p.part_A, place, w.lane, dA);
        }
    }
}

// dA, dskip, dbias: the parts of a channel block added up, always in the same order.  Workgroup (block, k):
// k < R S / 4: quads k of dA; k == R S / 4: the two vectors.  Wave w takes every fourth part.
template <int R, int S>
__global__ __launch_bounds__(256) void scan_sum_parts_kernel(ScanParams p) {
    constexpr int CH = 16 * R, QUADS = R * S / 4;
    __shared__ double sum[4][64][4];
    const int block = blockIdx.x / (QUADS + 1), k = blockIdx.x % (QUADS + 1);
    const int wave = threadIdx.x >> 6;
    const ScanLane<R, S> w(p, block);
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
__global__ __launch_bounds__(256) void scan_sum_bc_kernel(ScanParams p) {
    constexpr int NS = 4 * S;
    const int64_t first = min(max(p.off[0], (int64_t)0), p.frames);
    const int64_t last = min(max(p.off[p.utts], first), p.frames);
    const int64_t total = (last - first) * p.groups * 2 * NS;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int e = (int)(i % (2 * NS)), state = e % NS;
        const int64_t rest = i / (2 * NS);
        const int g = (int)(rest % p.groups);
        const int64_t t = first + rest / p.groups;
        float v = 0.0f;
        for (int k = 0; k < p.group_blocks; ++k)
            v += p.part_bc[((int64_t)(g * p.group_blocks + k) * p.frames + t) * 2 * NS + e];
        if (state < p.states) {
            const int64_t at = (int64_t)g * p.states + state;
            if (e < NS) ((T*)p.dB)[t * p.ld_dB + at] = (T)v;
            else ((T*)p.dC)[t * p.ld_dC + at] = (T)v;
        }
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
                v.v[k] = fmaf(exp_f32(d * a.v[k]), v.v[k], du * (float)b.v[k]);
                y = fmaf((float)q.v[k], v.v[k], y);
            }
            store_some(h + n0, v, left);
        }
        y += dpp_mov<0xB1>(y);       // quad_perm [1,0,3,2]
        y += dpp_mov<0x4E>(y);       // quad_perm [2,3,0,1]
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

template <typename T, int R, int S, bool GATE>
int scan_forward_launch(const ScanParams& p, hipStream_t st) {
    const int64_t across = (p.blocks + kScanWaves - 1) / kScanWaves;
    if (p.segment != 0) {
        scan_forward_kernel<T, R, S, GATE, 1><<<scan_grid(p.units * across), 64 * kScanWaves, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
        scan_join_kernel<R, S, false><<<scan_grid(p.utts * p.blocks), 64, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
    }
    scan_forward_kernel<T, R, S, GATE, 0><<<scan_grid(p.units * across), 64 * kScanWaves, 0, st>>>(p);
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

template <typename T, int R, int S, bool GATE>
int scan_backward_launch(const ScanParams& q, hipStream_t st) {
    ScanParams p = q;
    const int64_t across = (p.blocks + kScanWaves - 1) / kScanWaves;
    if (p.segment != 0) {
        const int64_t parts = p.parts;
        p.parts = p.units;
        scan_backward_kernel<T, R, S, GATE, 1><<<scan_grid(p.units * across), 64 * kScanWaves, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
        scan_join_kernel<R, S, true><<<scan_grid(p.utts * p.blocks), 64, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
        p.parts = parts;
    }
    scan_backward_kernel<T, R, S, GATE, 0><<<scan_grid(p.parts * across), 64 * kScanWaves, 0, st>>>(p);
    SRX_HIP(hipGetLastError());
    scan_sum_parts_kernel<R, S><<<(unsigned)(p.blocks * (R * S / 4 + 1)), 256, 0, st>>>(p);
    SRX_HIP(hipGetLastError());
    const int64_t sums = p.utts > 0 ? p.frames * p.groups * 8 * S : 0;
    if (sums > 0) {
        scan_sum_bc_kernel<T, S><<<scan_grid((sums + 255) / 256), 256, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
    }
    return SRX_OK;
}

template <typename T, bool GATE>
int scan_dispatch(const ScanParams& p, bool backward, hipStream_t st) {
#define SRX_SCAN_CASE(R, S)                                                                   \
    if (p.states <= 4 * S)                                                                    \
        return backward ? scan_backward_launch<T, R, S, GATE>(p, st) : scan_forward_launch<T, R, S, GATE>(p, st);
    SRX_SCAN_CASE(4, 1)
    SRX_SCAN_CASE(4, 2)
    SRX_SCAN_CASE(4, 4)
    SRX_SCAN_CASE(2, 8)
    SRX_SCAN_CASE(1, 16)
#undef SRX_SCAN_CASE
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
