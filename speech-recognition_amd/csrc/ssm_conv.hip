// Short causal convolution over the frames of each channel (srx_causal_conv): forward, backward and
// single-frame form.  Memory bound: a frame's element is read and written once, the filter's taps and the
// frames that it reaches back to stay in registers.  A thread owns neighbouring channels (one 16- or 8-byte
// access per frame) and walks over a piece of an utterance; neighbouring threads own neighbouring
// channels, so that a wave's access is one run of memory.  256 utterances of 100 to 300 frames x 2048 channels in
// bfloat16: 101 us, 4.2 TB/s; forward and backward of 64 x 1536 channels in float32: 30 (5.2 TB/s) and 53 us (4.4).
// Pieces of 64 frames and 16-byte accesses of 16-bit values, which leave fewer waves, are slower (110 us).
#include "frame_ops.h"

using namespace srx_frames;

namespace {

constexpr int kConvMaxWidth = 8;
constexpr int kConvPiece = 32;          // frames that a thread walks over

struct ConvParams {
    const float *weight, *bias;
    int channels, act;
    const int64_t* off;
    int64_t utts, frames;
    const void* x;
    int64_t ld_x;
    const void* state_in;
    void* state_out;
    void* y;
    int64_t ld_y;
    // backward
    const void* dy;
    int64_t ld_dy;
    const void* dstate_out;
    void* dx;
    int64_t ld_dx;
    void* dstate_in;
    float* part;            // [parts, width + 1, channels]
    int64_t parts;
    float *dweight, *dbias;
    int clear;              // workgroups (forward: rows of them) that set y's or dx's rows of no utterance to zero
};

struct ConvPiece {
    int64_t utt, begin, first, last, end;       // frames first .. last - 1 of begin .. end - 1
};

// Pieces are numbered off / kConvPiece + utterance + piece (see scan_unit in ssm_scan.h).
__device__ __forceinline__ bool conv_piece(const ConvParams& p, int64_t number, ConvPiece& w) {
    int64_t lo = 0, hi = p.utts - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        const int64_t at = min(max(p.off[mid], (int64_t)0), p.frames);
        if (at / kConvPiece + mid <= number) lo = mid;
        else hi = mid - 1;
    }
    const int64_t begin = min(max(p.off[lo], (int64_t)0), p.frames);
    const int64_t end = min(max(p.off[lo + 1], begin), p.frames);
    const int64_t piece = number - (begin / kConvPiece + lo);
    const int64_t first = begin + piece * kConvPiece;
    if (piece < 0 || (first >= end && piece > 0)) return false;
    w = {lo, begin, first, min(first + kConvPiece, end), end};
    return true;
}

template <typename T, int V, int W>
struct ConvTaps {
    float w[W][V], bias[V];
    __device__ __forceinline__ void load(const ConvParams& p, int c, int left) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            bias[v] = p.bias != nullptr && v < left ? p.bias[c + v] : 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][v] = v < left ? p.weight[(int64_t)(c + v) * W + k] : 0.0f;
        }
    }
    __device__ __forceinline__ void apply(const Pack<T, V> (&row)[W], float (&out)[V]) const {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s = bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) s = fmaf(w[k][v], (float)row[k].v[v], s);
            out[v] = s;
        }
    }
};

// Frame `place` (negative: before the utterance) of the piece's utterance.
template <typename T, int V, int W>
__device__ __forceinline__ Pack<T, V> conv_row(const ConvParams& p, const ConvPiece& w, int64_t place, int c, int left) {
    if (place >= 0) return load_some<V>((const T*)p.x + (w.begin + place) * p.ld_x + c, left);
    if (p.state_in == nullptr) {
        Pack<T, V> zero;
#pragma unroll
        for (int v = 0; v < V; ++v) zero.v[v] = (T)0.0f;
        return zero;
    }
    return load_some<V>((const T*)p.state_in + (w.utt * (W - 1) + place + W - 1) * p.channels + c, left);
}

// blockDim = (lanes, 256 / lanes), lanes across the channels; neighbouring workgroups have neighbouring channels, so that what
// runs at the same time covers whole rows and with them all memory channels.  A thread keeps its channels' taps over all the pieces
// that it takes.  The next four frames are on their way while four are computed.
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvParams p, int64_t pieces) {
    const int c = (int)(blockIdx.x * blockDim.x + threadIdx.x) * V, left = p.channels - c;
    const int groups = gridDim.y - p.clear;
    if ((int)blockIdx.y >= groups) {
        const int64_t group = (int64_t)(blockIdx.y - groups) * gridDim.x + blockIdx.x;
        clear_other_rows<T>(p.off, p.utts, p.frames, p.y, p.ld_y, p.channels, group * blockDim.y + threadIdx.y,
                            (int64_t)p.clear * gridDim.x * blockDim.y);
        return;
    }
    if (left <= 0) return;
    const bool all = (int)((blockIdx.x + 1) * blockDim.x) * V <= p.channels;      // (for the whole workgroup)
    ConvTaps<T, V, W> taps;
    taps.load(p, c, left);
    for (int64_t number = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; number < pieces;
         number += (int64_t)groups * blockDim.y) {
        ConvPiece w;
        if (!conv_piece(p, number, w)) continue;
        Pack<T, V> row[W];                       // the frames under the filter, oldest first
        constexpr int AHEAD = 4;
        Pack<T, V> in[AHEAD], next[AHEAD];
        const T* x = (const T*)p.x + c;
        if (w.first < w.last)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) next[i] = load_where<V>(all, x + min(w.first + i, w.last - 1) * p.ld_x, left);
        const int64_t place = w.first - w.begin;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) row[k + 1] = conv_row<T, V, W>(p, w, place - (W - 1) + k, c, left);
        // the state moves on here: this thread alone reads the old one, and has done so
        if (place == 0 && p.state_out != nullptr) {
            const int64_t length = w.end - w.begin;
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                Pack<T, V> v;
                if (length + j >= W - 1) {
                    v = conv_row<T, V, W>(p, w, length - (W - 1) + j, c, left);
                } else {
#pragma unroll
                    for (int k = 0; k < W - 1; ++k)
                        if (k == length + j) v = row[k + 1];
                }
                store_some((T*)p.state_out + (w.utt * (W - 1) + j) * p.channels + c, v, left);
            }
        }
        for (int64_t t0 = w.first; t0 < w.last; t0 += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) in[i] = next[i];
            if (t0 + AHEAD < w.last)
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    next[i] = load_where<V>(all, x + min(t0 + AHEAD + i, w.last - 1) * p.ld_x, left);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k) row[k] = row[k + 1];
                row[W - 1] = in[i];
                float s[V];
                taps.apply(row, s);
                Pack<T, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) out.v[v] = (T)(p.act == SRX_SILU ? s[v] * sigmoid_f32(s[v]) : s[v]);
                if (t0 + i < w.last) store_where(all, (T*)p.y + (t0 + i) * p.ld_y + c, out, left);
            }
        }
    }
}

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvParams p, int64_t rows, int vectors) {
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < rows * vectors; id += (int64_t)gridDim.x * 256) {
        const int64_t u = id / vectors;
        const int c = (int)(id - u * vectors) * V, left = p.channels - c;
        ConvTaps<T, V, W> taps;
        taps.load(p, c, left);
        T* state = (T*)p.state_out + u * (W - 1) * p.channels + c;
        Pack<T, V> row[W];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) row[k] = load_some<V>(state + (int64_t)k * p.channels, left);
        row[W - 1] = load_some<V>((const T*)p.x + u * p.ld_x + c, left);
        float s[V];
        taps.apply(row, s);
        Pack<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) out.v[v] = (T)(p.act == SRX_SILU ? s[v] * sigmoid_f32(s[v]) : s[v]);
        store_some((T*)p.y + u * p.ld_y + c, out, left);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) store_some(state + (int64_t)k * p.channels, row[k + 1], left);
    }
}

// dx[t] = sum_k w[k] g[t + width - 1 - k] with g = dy act'(s); the sum s is computed again from x.  A
// thread walks over its piece and the width - 1 frames behind it, whose g reach back into the piece.  The
// taps' gradients are summed in registers over the pieces that a workgroup takes, joined through LDS, and
// written as one part per workgroup.  blockDim = (lanes, 256 / lanes): lanes across the channels.
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvParams p, int64_t pieces) {
    __shared__ float sums[256 * (W + 1) * V];
    const int c = (int)(blockIdx.x * blockDim.x + threadIdx.x) * V, left = p.channels - c;
    const bool all = (int)((blockIdx.x + 1) * blockDim.x) * V <= p.channels;      // (for the whole workgroup)
    ConvTaps<T, V, W> taps;
    taps.load(p, c, left);
    float dw[W][V], db[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][v] = 0.0f;
    }
    for (int64_t number = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; number < pieces;
         number += (int64_t)gridDim.y * blockDim.y) {
        ConvPiece w;
        if (left <= 0 || !conv_piece(p, number, w)) continue;
        const int64_t place = w.first - w.begin, length = w.end - w.begin;
        Pack<T, V> row[W];
        float g[W][V];                            // of the last W frames, oldest first
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) g[k][v] = 0.0f;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) row[k + 1] = conv_row<T, V, W>(p, w, place - (W - 1) + k, c, left);
        const int64_t stop = w.last + W - 1;      // frames past the utterance's end have g = 0
        constexpr int AHEAD = 4;
        for (int64_t t0 = w.first; t0 < stop; t0 += AHEAD) {
            Pack<T, V> in[AHEAD], dy[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int64_t t = min(t0 + i, w.end - 1);
                if (w.end > w.begin) {
                    in[i] = load_where<V>(all, (const T*)p.x + t * p.ld_x + c, left);
                    dy[i] = load_where<V>(all, (const T*)p.dy + t * p.ld_dy + c, left);
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int64_t t = t0 + i;
                if (t >= stop) break;
#pragma unroll
                for (int k = 0; k < W - 1; ++k) row[k] = row[k + 1];
                row[W - 1] = in[i];
#pragma unroll
                for (int k = 0; k < W - 1; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v) g[k][v] = g[k + 1][v];
                if (t < w.end) {
                    float s[V];
                    taps.apply(row, s);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        float d = (float)dy[i].v[v];
                        if (p.act == SRX_SILU) {
                            const float sig = sigmoid_f32(s[v]);
                            d *= sig * fmaf(s[v], 1.0f - sig, 1.0f);
                        }
                        g[W - 1][v] = d;
                        if (t < w.last) {
                            db[v] += d;
#pragma unroll
                            for (int k = 0; k < W; ++k) dw[k][v] = fmaf(d, (float)row[k].v[v], dw[k][v]);
                        }
                    }
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) g[W - 1][v] = 0.0f;
                }
                // frame t - (W - 1), of this piece or, at its head, of the state
                const int64_t at = t - (W - 1) - w.begin;       // place in the utterance
                const bool own = t - (W - 1) >= w.first;
                if (!own && (place != 0 || p.dstate_in == nullptr)) continue;
                Pack<T, V> out;
                float d[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    d[v] = 0.0f;
#pragma unroll
                    for (int k = 0; k < W; ++k) d[v] = fmaf(taps.w[k][v], g[W - 1 - k][v], d[v]);
                }
                const int64_t kept = at - (length - (W - 1));   // its row of the outgoing state
                if (p.dstate_out != nullptr && kept >= 0) {
                    const Pack<T, V> more = load_some<V>((const T*)p.dstate_out + (w.utt * (W - 1) + kept) * p.channels + c, left);
#pragma unroll
                    for (int v = 0; v < V; ++v) d[v] += (float)more.v[v];
                }
#pragma unroll
                for (int v = 0; v < V; ++v) out.v[v] = (T)d[v];
                if (own) store_where(all, (T*)p.dx + (t - (W - 1)) * p.ld_dx + c, out, left);
                else store_some((T*)p.dstate_in + (w.utt * (W - 1) + at + W - 1) * p.channels + c, out, left);
            }
        }
    }
    // join the workgroup's rows of threads
    const int lanes = blockDim.x;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < W; ++k) sums[((threadIdx.y * (W + 1) + k) * lanes + threadIdx.x) * V + v] = dw[k][v];
        sums[((threadIdx.y * (W + 1) + W) * lanes + threadIdx.x) * V + v] = db[v];
    }
    __syncthreads();
    const int wide = lanes * V;
    for (int e = threadIdx.y * lanes + threadIdx.x; e < (W + 1) * wide; e += 256) {
        const int k = e / wide, at = e - k * wide, channel = (int)blockIdx.x * wide + at;
        float s = 0.0f;
        for (int y = 0; y < (int)blockDim.y; ++y) s += sums[(y * (W + 1) + k) * wide + at];
        if (channel < p.channels) p.part[((int64_t)blockIdx.y * (W + 1) + k) * p.channels + channel] = s;
    }
}

template <typename T>
__global__ __launch_bounds__(kSumThreads) void conv_sum_kernel(ConvParams p, int width) {
    const int groups = gridDim.x - p.clear;
    if ((int)blockIdx.x >= groups) {             // (the gradients of frames that belong to no utterance)
        clear_other_rows<T>(p.off, p.utts, p.frames, p.dx, p.ld_dx, p.channels, blockIdx.x - groups, p.clear);
        return;
    }
    sum_parts(p.part, p.parts, (int64_t)(width + 1) * p.channels, [&](int64_t column, double s) {
        const int k = (int)(column / p.channels), c = (int)(column - (int64_t)k * p.channels);
        if (k < width) p.dweight[(int64_t)c * width + k] = (float)s;
        else if (p.dbias != nullptr) p.dbias[c] = (float)s;
    });
}

constexpr int64_t kMostWorkgroups = 1 << 22;
unsigned conv_grid(int64_t threads) {
    const int64_t n = (threads + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n < kMostWorkgroups ? n : kMostWorkgroups);
}

int64_t conv_pieces(int64_t utts, int64_t frames) { return utts == 0 ? 0 : frames / kConvPiece + utts; }

constexpr int kBackwardVector = 4;
constexpr int kForwardVector = 4;
constexpr int kClearRows = 16;          // of workgroups, for rows of no utterance

int conv_lanes(int channels, int v) {
    const int vectors = (channels + v - 1) / v;
    int lanes = 8;
    while (lanes < 64 && lanes < vectors) lanes *= 2;
    return lanes;
}
// Workgroups along the pieces: enough to fill the chip several times over, and few enough frames per thread
// that the 32-bit sums of the taps' gradients stay exact to a few units of rounding.  (Beyond what a grid's second
// dimension has room for, 130 million frames at the least, the sums get longer.)
constexpr int kConvMostSummed = 512;
int64_t conv_parts(const srx_context* h, int channels, int64_t utts, int64_t frames) {
    const int lanes = conv_lanes(channels, kBackwardVector), rows = 256 / lanes;
    const int64_t across = (channels + lanes * kBackwardVector - 1) / (lanes * kBackwardVector);
    const int64_t groups = (conv_pieces(utts, frames) + rows - 1) / rows;
    const int64_t fill = ((int64_t)h->n_cu * 8 + across - 1) / across;
    constexpr int64_t most = kConvMostSummed / kConvPiece;
    const int64_t exact = (groups + most - 1) / most;
    const int64_t parts = groups < fill ? groups : fill > exact ? fill : exact;
    return parts < 1 ? 1 : parts < 65535 ? parts : 65535;              // (a grid's second dimension)
}

enum ConvWhat { FORWARD, STEP, BACKWARD };

template <typename T, int W>
int conv_launch(const ConvParams& p, ConvWhat what, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int vectors = (p.channels + V - 1) / V;
    const int64_t pieces = conv_pieces(p.utts, p.frames);
    if (what == STEP) {
        conv_step_kernel<T, V, W><<<conv_grid(p.utts * vectors), 256, 0, st>>>(p, p.utts, vectors);
    } else if (what == FORWARD) {
        constexpr int FV = kForwardVector;
        const int lanes = conv_lanes(p.channels, FV), rows = 256 / lanes;
        const int64_t across = (p.channels + lanes * FV - 1) / (lanes * FV), groups = (pieces + rows - 1) / rows;
        const int64_t fill = (p.parts + across - 1) / across;       // (parts: the workgroups that the chip holds)
        conv_forward_kernel<T, FV, W><<<dim3((unsigned)across, (unsigned)(groups < fill ? groups : fill) + p.clear), dim3(lanes, rows), 0, st>>>(p, pieces);
    } else {
        const int lanes = conv_lanes(p.channels, kBackwardVector);
        const int across = (p.channels + lanes * kBackwardVector - 1) / (lanes * kBackwardVector);
        conv_backward_kernel<T, kBackwardVector, W><<<dim3((unsigned)across, (unsigned)p.parts), dim3(lanes, 256 / lanes), 0, st>>>(p, pieces);
        SRX_HIP(hipGetLastError());
        conv_sum_kernel<T><<<((W + 1) * p.channels + 31) / 32 + p.clear, kSumThreads, 0, st>>>(p, W);
    }
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

template <typename T>
int conv_width(const ConvParams& p, int width, ConvWhat what, hipStream_t st) {
    switch (width) {
        case 1: return conv_launch<T, 1>(p, what, st);
        case 2: return conv_launch<T, 2>(p, what, st);
        case 3: return conv_launch<T, 3>(p, what, st);
        case 4: return conv_launch<T, 4>(p, what, st);
        case 5: return conv_launch<T, 5>(p, what, st);
        case 6: return conv_launch<T, 6>(p, what, st);
        case 7: return conv_launch<T, 7>(p, what, st);
        default: return conv_launch<T, 8>(p, what, st);
    }
}

int conv_run(const ConvParams& p, int width, int dtype, ConvWhat what, hipStream_t st) {
    switch (dtype) {
        case SRX_F32: return conv_width<float>(p, width, what, st);
        case SRX_BF16: return conv_width<__bf16>(p, width, what, st);
        default: return conv_width<_Float16>(p, width, what, st);
    }
}

int check_conv(srx_handle_t h, const srx_conv_t* conv, int64_t utts, int64_t frames, const char* who) {
    SRX_REQUIRE(h != nullptr, "%s: NULL context", who);
    SRX_REQUIRE(conv != nullptr, "%s: conv is NULL", who);
    SRX_REQUIRE(conv->n_channels >= 1, "%s: Shape mismatch (n_channels=%d)", who, conv->n_channels);
    SRX_REQUIRE(conv->n_channels <= kMostColumns, "%s: n_channels %d above 2^24", who, conv->n_channels);
    SRX_REQUIRE(conv->width >= 1 && conv->width <= kConvMaxWidth, "%s: width %d outside [1, %d]", who, conv->width,
                kConvMaxWidth);
    SRX_REQUIRE(conv->activation == SRX_IDENTITY || conv->activation == SRX_SILU, "%s: unknown activation %d", who,
                conv->activation);
    SRX_REQUIRE(conv->weight != nullptr, "%s: NULL weight", who);
    SRX_REQUIRE(utts >= 0 && frames >= 0, "%s: negative size", who);
    return SRX_OK;
}

ConvParams conv_params(const srx_conv_t* conv, const int64_t* off, int64_t utts, int64_t frames, const void* x, int64_t ld_x) {
    ConvParams p;
    memset(&p, 0, sizeof(p));
    p.weight = conv->weight;
    p.bias = conv->bias;
    p.channels = conv->n_channels;
    p.act = conv->activation;
    p.off = off;
    p.utts = utts;
    p.frames = frames;
    p.x = x;
    p.ld_x = ld_x;
    return p;
}

}  // namespace

extern "C" {

int srx_causal_conv(srx_handle_t h, const srx_conv_t* conv, int dtype, const void* x, int64_t ld_x,
                    const int64_t* utt_offsets, int64_t n_utts, int64_t n_frames, const void* state_in,
                    void* state_out, void* y, int64_t ld_y, void* stream) {
    const char* who = "srx_causal_conv";
    const bool zero = take_zero_rows(dtype) && n_frames > 0;
    int rc = check_conv(h, conv, n_utts, n_frames, who);
    if (rc) return rc;
    SRX_REQUIRE(frame_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    if (n_utts == 0 && !zero) return SRX_OK;
    SRX_REQUIRE(n_utts == 0 || utt_offsets != nullptr, "%s: NULL utterance offsets", who);
    SRX_REQUIRE(n_frames == 0 || (x != nullptr && y != nullptr), "%s: NULL x or y", who);
    SRX_REQUIRE(n_frames == 0 || (ld_x >= conv->n_channels && ld_y >= conv->n_channels),
                "%s: a row pitch is smaller than its row", who);
    ConvParams p = conv_params(conv, utt_offsets, n_utts, n_frames, x, ld_x);
    p.state_in = state_in;
    p.state_out = state_out;
    p.y = y;
    p.ld_y = ld_y;
    p.parts = (int64_t)h->n_cu * 16;
    p.clear = zero ? kClearRows : 0;
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return conv_run(p, conv->width, dtype, FORWARD, (hipStream_t)stream);
}

int srx_causal_conv_step(srx_handle_t h, const srx_conv_t* conv, int dtype, const void* x, int64_t ld_x,
                         int64_t n_rows, void* state, void* y, int64_t ld_y, void* stream) {
    const char* who = "srx_causal_conv_step";
    int rc = check_conv(h, conv, n_rows, n_rows, who);
    if (rc) return rc;
    SRX_REQUIRE(frame_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    if (n_rows == 0) return SRX_OK;
    SRX_REQUIRE(x != nullptr && y != nullptr && (state != nullptr || conv->width == 1), "%s: NULL x, y or state", who);
    SRX_REQUIRE(ld_x >= conv->n_channels && ld_y >= conv->n_channels, "%s: a row pitch is smaller than its row", who);
    ConvParams p = conv_params(conv, nullptr, n_rows, n_rows, x, ld_x);
    p.state_out = state;
    p.y = y;
    p.ld_y = ld_y;
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return conv_run(p, conv->width, dtype, STEP, (hipStream_t)stream);
}

int64_t srx_causal_conv_backward_workspace(srx_handle_t h, const srx_conv_t* conv, int64_t n_utts, int64_t n_frames) {
    if (check_conv(h, conv, n_utts, n_frames, "srx_causal_conv_backward_workspace")) return -1;
    return conv_parts(h, conv->n_channels, n_utts, n_frames) * (conv->width + 1) * conv->n_channels * 4;
}

int srx_causal_conv_backward(srx_handle_t h, const srx_conv_t* conv, int dtype, const void* x, int64_t ld_x,
                             const int64_t* utt_offsets, int64_t n_utts, int64_t n_frames, const void* state_in,
                             const void* dy, int64_t ld_dy, const void* dstate_out, void* dx, int64_t ld_dx,
                             float* dweight, float* dbias, void* dstate_in, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    const char* who = "srx_causal_conv_backward";
    int rc = check_conv(h, conv, n_utts, n_frames, who);
    if (rc) return rc;
    SRX_REQUIRE(frame_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    SRX_REQUIRE(n_utts == 0 || utt_offsets != nullptr, "%s: NULL utterance offsets", who);
    SRX_REQUIRE(dweight != nullptr, "%s: NULL dweight", who);
    SRX_REQUIRE(n_frames == 0 || (x != nullptr && dy != nullptr && dx != nullptr), "%s: NULL x, dy or dx", who);
    SRX_REQUIRE(n_frames == 0 || (ld_x >= conv->n_channels && ld_dy >= conv->n_channels && ld_dx >= conv->n_channels),
                "%s: a row pitch is smaller than its row", who);
    const int64_t need = srx_causal_conv_backward_workspace(h, conv, n_utts, n_frames);
    SRX_REQUIRE(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %lld bytes, %lld are needed", who,
                (long long)workspace_bytes, (long long)need);
    ConvParams p = conv_params(conv, utt_offsets, n_utts, n_frames, x, ld_x);
    p.state_in = state_in;
    p.dy = dy;
    p.ld_dy = ld_dy;
    p.dstate_out = dstate_out;
    p.dx = dx;
    p.ld_dx = ld_dx;
    p.dstate_in = dstate_in;
    p.dweight = dweight;
    p.dbias = dbias;
    p.clear = n_frames > 0 ? kClearGroups : 0;
    p.part = (float*)workspace;
    p.parts = conv_parts(h, conv->n_channels, n_utts, n_frames);
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return conv_run(p, conv->width, dtype, BACKWARD, (hipStream_t)stream);
}

}  // extern "C"
