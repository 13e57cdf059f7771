// Layer norm of frames (srx_layer_norm): forward and backward with the weights' gradients.  Memory bound.
// A row is held in registers by 16 or 64 lanes of a wave or by a whole workgroup, by its width, and read
// once: mean first, then the squares of what is left, so that a mean far from zero costs no accuracy.
// Wider rows than a workgroup's registers hold are read again for each of the passes.  65,536 rows of 1024 values in
// bfloat16: forward 55 us, backward 83 us, 4.9 TB/s; 1,310,720 rows of 39 in float32: 85 us, 4.8 TB/s.
// Slower: the backward pass of narrow rows (1,310,720 of 39: 153 us, 4.0 TB/s, in bfloat16 159 us, 1.9), and rows above 4096
// (6000 of 8192 in float32: 148 and 419 us, 2.7 and 1.4 TB/s).
#include "frame_ops.h"

using namespace srx_frames;

namespace {

struct NormParams {
    const void* x;
    int64_t ld_x;
    int64_t rows;
    int width;
    const float *weight, *bias;
    float eps;
    void* y;
    int64_t ld_y;
    float *mean, *rstd;
    const void* dy;
    int64_t ld_dy;
    void* dx;
    int64_t ld_dx;
    float *dweight, *dbias;
    float* part;                // [parts, 2, width]
    int64_t parts;
};

// Sums over the lanes that share a row, in all of them.
template <int LANES>
__device__ __forceinline__ void row_sums(float& a, float& b, float* shared) {
    a = row16_sum(a);
    b = row16_sum(b);
    if constexpr (LANES >= 64) {
        a = rows_sum(a, a);
        b = rows_sum(b, b);
        a = halves_sum(a, a);
        b = halves_sum(b, b);
    }
    if constexpr (LANES == 256) {
        __syncthreads();                          // (the last sums have been read)
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            shared[wave] = a;
            shared[4 + wave] = b;
        }
        __syncthreads();
        a = (shared[0] + shared[1]) + (shared[2] + shared[3]);
        b = (shared[4] + shared[5]) + (shared[6] + shared[7]);
    }
}

// Column of element v of vector k of a lane.
template <int LANES, int V>
__device__ __forceinline__ int norm_column(int lane, int k) { return (k * LANES + lane) * V; }

template <typename T, int LANES, int NV, int V>
__global__ __launch_bounds__(256) void norm_forward_kernel(NormParams p) {
    __shared__ float shared[8];
    constexpr int ROWS = 256 / LANES;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float n = (float)p.width;
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = norm_column<LANES, V>(lane, k) + v;
            w[k][v] = p.weight != nullptr && c < p.width ? p.weight[c] : 1.0f;
            b[k][v] = p.bias != nullptr && c < p.width ? p.bias[c] : 0.0f;
        }
    // (a workgroup's threads leave the loop together where they share a row)
    for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < p.rows; row += (int64_t)gridDim.x * ROWS) {
        const T* x = (const T*)p.x + row * p.ld_x;
        float f[NV][V], sum = 0.0f, none = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = norm_column<LANES, V>(lane, k);
            const Pack<T, V> in = load_where<V>((k + 1) * LANES * V <= p.width, x + c, p.width - c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[k][v] = (float)in.v[v];
                sum += f[k][v];
            }
        }
        row_sums<LANES>(sum, none, shared);
        const float mean = sum / n;
        float square = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const bool in = norm_column<LANES, V>(lane, k) + v < p.width;
                f[k][v] = in ? f[k][v] - mean : 0.0f;
                square = fmaf(f[k][v], f[k][v], square);
            }
        row_sums<LANES>(square, none, shared);
        const float rstd = 1.0f / sqrtf(square / n + p.eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = norm_column<LANES, V>(lane, k);
            Pack<T, V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) out.v[v] = (T)fmaf(f[k][v] * rstd, w[k][v], b[k][v]);
            store_where((k + 1) * LANES * V <= p.width, (T*)p.y + row * p.ld_y + c, out, p.width - c);
        }
        if (lane == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

// dx = rstd (g - mean(g) - xhat mean(g xhat)), g = dy weight; the rows that a lane meets are summed
// into its columns of dweight and dbias, one part per workgroup.
template <typename T, int LANES, int NV, int V>
__global__ __launch_bounds__(256) void norm_backward_kernel(NormParams p) {
    constexpr int ROWS = 256 / LANES, WIDE = LANES * NV * V;
    __shared__ float shared[ROWS > 1 ? ROWS * WIDE : 8];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float share = 1.0f / (float)p.width;
    float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = norm_column<LANES, V>(lane, k) + v;
            w[k][v] = p.weight != nullptr && c < p.width ? p.weight[c] : 1.0f;
            dw[k][v] = db[k][v] = 0.0f;
        }
    for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < p.rows; row += p.parts * ROWS) {
        const T* x = (const T*)p.x + row * p.ld_x;
        const T* dy = (const T*)p.dy + row * p.ld_dy;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float unit[NV][V], g[NV][V], a = 0.0f, b = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = norm_column<LANES, V>(lane, k);
            const bool all = (k + 1) * LANES * V <= p.width;
            const Pack<T, V> in = load_where<V>(all, x + c, p.width - c), d = load_where<V>(all, dy + c, p.width - c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float dv = (float)d.v[v];
                unit[k][v] = c + v < p.width ? ((float)in.v[v] - mean) * rstd : 0.0f;
                g[k][v] = dv * w[k][v];
                dw[k][v] = fmaf(dv, unit[k][v], dw[k][v]);
                db[k][v] += dv;
                a += g[k][v];
                b = fmaf(g[k][v], unit[k][v], b);
            }
        }
        row_sums<LANES>(a, b, shared);
        a *= share;
        b *= share;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = norm_column<LANES, V>(lane, k);
            Pack<T, V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) out.v[v] = (T)(rstd * (g[k][v] - a - unit[k][v] * b));
            store_where((k + 1) * LANES * V <= p.width, (T*)p.dx + row * p.ld_dx + c, out, p.width - c);
        }
    }
    // the rows of threads joined, dweight first and dbias after it in the same memory
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* part = p.part + ((int64_t)blockIdx.x * 2 + which) * p.width;
        if constexpr (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    shared[sub * WIDE + norm_column<LANES, V>(lane, k) + v] = which ? db[k][v] : dw[k][v];
            __syncthreads();
            for (int c = threadIdx.x; c < p.width; c += 256) {
                float s = 0.0f;
#pragma unroll
                for (int r = 0; r < ROWS; ++r) s += shared[r * WIDE + c];
                part[c] = s;
            }
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int c = norm_column<LANES, V>(lane, k) + v;
                    if (c < p.width) part[c] = which ? db[k][v] : dw[k][v];
                }
        }
    }
}

// Rows wider than a workgroup's registers: one workgroup per row, three passes over it.
template <typename T>
__global__ __launch_bounds__(256) void norm_forward_wide_kernel(NormParams p) {
    __shared__ float shared[8];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ld_x;
        float sum = 0.0f, square = 0.0f, none = 0.0f;
        for (int c = threadIdx.x; c < p.width; c += 256) sum += (float)x[c];
        row_sums<256>(sum, none, shared);
        const float mean = sum / (float)p.width;
        for (int c = threadIdx.x; c < p.width; c += 256) {
            const float d = (float)x[c] - mean;
            square = fmaf(d, d, square);
        }
        row_sums<256>(square, none, shared);
        const float rstd = 1.0f / sqrtf(square / (float)p.width + p.eps);
        for (int c = threadIdx.x; c < p.width; c += 256) {
            const float w = p.weight != nullptr ? p.weight[c] : 1.0f, b = p.bias != nullptr ? p.bias[c] : 0.0f;
            ((T*)p.y)[row * p.ld_y + c] = (T)fmaf(((float)x[c] - mean) * rstd, w, b);
        }
        if (threadIdx.x == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void norm_backward_wide_kernel(NormParams p) {
    __shared__ float shared[8];
    float* dw = p.part + (int64_t)blockIdx.x * 2 * p.width;
    float* db = dw + p.width;
    for (int c = threadIdx.x; c < p.width; c += 256) dw[c] = db[c] = 0.0f;      // (each thread its own columns)
    for (int64_t row = blockIdx.x; row < p.rows; row += p.parts) {
        const T* x = (const T*)p.x + row * p.ld_x;
        const T* dy = (const T*)p.dy + row * p.ld_dy;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float a = 0.0f, b = 0.0f;
        for (int c = threadIdx.x; c < p.width; c += 256) {
            const float d = (float)dy[c], unit = ((float)x[c] - mean) * rstd;
            const float g = d * (p.weight != nullptr ? p.weight[c] : 1.0f);
            dw[c] = fmaf(d, unit, dw[c]);
            db[c] += d;
            a += g;
            b = fmaf(g, unit, b);
        }
        row_sums<256>(a, b, shared);
        a /= (float)p.width;
        b /= (float)p.width;
        for (int c = threadIdx.x; c < p.width; c += 256) {
            const float unit = ((float)x[c] - mean) * rstd;
            const float g = (float)dy[c] * (p.weight != nullptr ? p.weight[c] : 1.0f);
            ((T*)p.dx)[row * p.ld_dx + c] = (T)(rstd * (g - a - unit * b));
        }
    }
}

__global__ __launch_bounds__(kSumThreads) void norm_sum_kernel(NormParams p) {
    sum_parts(p.part, p.parts, 2 * (int64_t)p.width, [&](int64_t column, double s) {
        float* to = column < p.width ? p.dweight : p.dbias;
        if (to != nullptr) to[column < p.width ? column : column - p.width] = (float)s;
    });
}

// Narrow rows (the front-end's features): a workgroup takes 128 of them into LDS -- as one run of memory where there
// are no gaps between them --, each thread then has a row of its own in registers and needs no other lane for its
// sums, and the results leave the same way.  An odd distance between the rows in LDS keeps 64 threads on 64 banks; rows of
// an odd width lie there as in memory and are moved 16 bytes at a time.  EIGHTS: of the row's values, rounded up.
constexpr int kNarrowRows = 128;

// Calls each(element, place) for the next V elements of a run of whole rows, from element e on.
template <int V, typename F>
__device__ __forceinline__ void narrow_places(int e, int width, int step, const F& each) {
    int r = e / width, c = e - r * width;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        each(v, r * step + c);
        if (++c == width) {
            c = 0;
            ++r;
        }
    }
}

template <typename T, int EIGHTS>
__global__ __launch_bounds__(kNarrowRows) void norm_forward_narrow_kernel(NormParams p) {
    constexpr int V = 16 / sizeof(T), RUN = kNarrowRows * V, AHEAD = sizeof(T), WIDE = 8 * EIGHTS;
    extern __shared__ __align__(16) float rows[];              // [128][width | 1], weight and bias after them
    const int width = p.width, step = width | 1;
    const bool odd = step == width;
    float* weight = rows + kNarrowRows * step;
    float* bias = weight + WIDE;
    for (int c = threadIdx.x; c < width; c += kNarrowRows) {
        weight[c] = p.weight != nullptr ? p.weight[c] : 1.0f;
        bias[c] = p.bias != nullptr ? p.bias[c] : 0.0f;
    }
    for (int64_t row0 = (int64_t)blockIdx.x * kNarrowRows; row0 < p.rows; row0 += (int64_t)gridDim.x * kNarrowRows) {
        const int here = (int)min((int64_t)kNarrowRows, p.rows - row0), count = here * width;
        __syncthreads();                         // (the last rows have left)
        if (p.ld_x != width) {
            for (int e = threadIdx.x; e < count; e += kNarrowRows) {
                const int r = e / width, c = e - r * width;
                rows[r * step + c] = (float)((const T*)p.x)[(row0 + r) * p.ld_x + c];
            }
        } else {
            const T* x = (const T*)p.x + row0 * width;
            for (int first = 0; first < count; first += AHEAD * RUN) {
                Pack<T, V> in[AHEAD];            // (several on their way at once)
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int e = first + k * RUN + threadIdx.x * V;
                    in[k] = load_where<V>(first + (k + 1) * RUN <= count, x + e, count - e);
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int e = first + k * RUN + threadIdx.x * V;
                    if (odd) {
                        Pack<float, V> f;
#pragma unroll
                        for (int v = 0; v < V; ++v) f.v[v] = (float)in[k].v[v];
                        store_where(first + (k + 1) * RUN <= count, rows + e, f, count - e);
                    } else {
                        narrow_places<V>(e, width, step, [&](int v, int at) {
                            if (e + v < count) rows[at] = (float)in[k].v[v];
                        });
                    }
                }
            }
        }
        __syncthreads();
        if ((int)threadIdx.x < here) {
            float* mine = rows + threadIdx.x * step;
            float f[WIDE], sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < WIDE; ++c) {
                const bool in = c < WIDE - 8 || c < width;
                f[c] = in ? mine[c] : 0.0f;
                sum[c % 4] += f[c];
            }
            const float mean = ((sum[0] + sum[1]) + (sum[2] + sum[3])) / (float)width;
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = 0.0f;
#pragma unroll
            for (int c = 0; c < WIDE; ++c) {
                f[c] = c < WIDE - 8 || c < width ? f[c] - mean : 0.0f;
                sum[c % 4] = fmaf(f[c], f[c], sum[c % 4]);
            }
            const float rstd = 1.0f / sqrtf(((sum[0] + sum[1]) + (sum[2] + sum[3])) / (float)width + p.eps);
#pragma unroll
            for (int c = 0; c < WIDE; c += 4) {
                const Pack<float, 4> w = load_pack<4>(weight + c), b = load_pack<4>(bias + c);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (c + k < WIDE - 8 || c + k < width) mine[c + k] = fmaf(f[c + k] * rstd, w.v[k], b.v[k]);
            }
            p.mean[row0 + threadIdx.x] = mean;
            p.rstd[row0 + threadIdx.x] = rstd;
        }
        __syncthreads();
        if (p.ld_y != width) {
            for (int e = threadIdx.x; e < count; e += kNarrowRows) {
                const int r = e / width, c = e - r * width;
                ((T*)p.y)[(row0 + r) * p.ld_y + c] = (T)rows[r * step + c];
            }
        } else {
            T* y = (T*)p.y + row0 * width;
            for (int first = 0; first < count; first += RUN) {
                const int e = first + threadIdx.x * V;
                Pack<T, V> out;
                if (odd) {
                    const Pack<float, V> f = load_where<V>(first + RUN <= count, (const float*)rows + e, count - e);
#pragma unroll
                    for (int v = 0; v < V; ++v) out.v[v] = (T)f.v[v];
                } else {
                    narrow_places<V>(e, width, step, [&](int v, int at) { out.v[v] = (T)(e + v < count ? rows[at] : 0.0f); });
                }
                store_where(first + RUN <= count, y + e, out, count - e);
            }
        }
    }
}

// How a row is held: lanes, vectors per lane; lanes 0: not in registers.
struct NormShape {
    int lanes, vectors;
};
NormShape norm_shape(int width, int v) {
    const NormShape shapes[] = {{16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}};
    for (const NormShape& s : shapes)
        if (width <= s.lanes * s.vectors * v) return s;
    return {0, 0};
}

int64_t norm_parts(const srx_context* h, int64_t rows, int width) {
    const NormShape s = norm_shape(width, 4);
    const int per = s.lanes == 0 ? 1 : 256 / s.lanes;
    const int64_t groups = (rows + per - 1) / per;
    // four workgroups per CU, and at most 256 rows per thread so that its 32-bit sums stay exact to a few
    // units of rounding
    const int64_t fill = (int64_t)h->n_cu * 4, exact = (groups + 255) / 256;
    const int64_t parts = groups < fill ? groups : fill > exact ? fill : exact;
    return parts < 1 ? 1 : parts;
}

template <typename T, int LANES, int NV, int V>
int norm_go(const NormParams& p, bool backward, hipStream_t st) {
    constexpr int ROWS = 256 / LANES;
    if (backward) {
        norm_backward_kernel<T, LANES, NV, V><<<(unsigned)p.parts, 256, 0, st>>>(p);
    } else {
        // (a workgroup keeps weight and bias over its rows)
        const int64_t groups = (p.rows + ROWS - 1) / ROWS, most = p.parts;
        norm_forward_kernel<T, LANES, NV, V><<<(unsigned)(groups < most ? groups : most), 256, 0, st>>>(p);
    }
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

template <typename T, int EIGHTS>
int norm_narrow(const NormParams& p, hipStream_t st) {
    const int64_t groups = (p.rows + kNarrowRows - 1) / kNarrowRows;
    const size_t lds = (size_t)(kNarrowRows * (p.width | 1) + 16 * EIGHTS) * sizeof(float);
    norm_forward_narrow_kernel<T, EIGHTS><<<(unsigned)(groups < 2 * p.parts ? groups : 2 * p.parts), kNarrowRows, lds, st>>>(p);
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

template <typename T>
int norm_typed(const NormParams& p, bool backward, hipStream_t st) {
    const NormShape s = norm_shape(p.width, 4);
    // Narrow rows (1,000,000 of them in float32, 16 lanes per row against one thread): 16 values 54 us and 26, 32 55 and
    // 51, 40 67 and 78; odd widths, whose rows those lanes load value by value, 39 107 and 66, 63 137 and 111.
    if (!backward && (p.width <= 32 || (p.width < 64 && p.width % 2 == 1))) {
        switch ((p.width + 7) / 8) {
            case 1: return norm_narrow<T, 1>(p, st);
            case 2: return norm_narrow<T, 2>(p, st);
            case 3: return norm_narrow<T, 3>(p, st);
            case 4: return norm_narrow<T, 4>(p, st);
            case 5: return norm_narrow<T, 5>(p, st);
            case 6: return norm_narrow<T, 6>(p, st);
            case 7: return norm_narrow<T, 7>(p, st);
            default: return norm_narrow<T, 8>(p, st);
        }
    }
    if (s.lanes == 16 && s.vectors == 1) return norm_go<T, 16, 1, 4>(p, backward, st);
    if (s.lanes == 16) return norm_go<T, 16, 2, 4>(p, backward, st);
    if (s.lanes == 64 && s.vectors == 1) return norm_go<T, 64, 1, 4>(p, backward, st);
    if (s.lanes == 64 && s.vectors == 2) return norm_go<T, 64, 2, 4>(p, backward, st);
    if (s.lanes == 64) return norm_go<T, 64, 4, 4>(p, backward, st);
    if (s.lanes == 256 && s.vectors == 2) return norm_go<T, 256, 2, 4>(p, backward, st);
    if (s.lanes == 256) return norm_go<T, 256, 4, 4>(p, backward, st);
    if (backward) {
        norm_backward_wide_kernel<T><<<(unsigned)p.parts, 256, 0, st>>>(p);
    } else {
        norm_forward_wide_kernel<T><<<(unsigned)(p.rows < (1 << 20) ? p.rows : 1 << 20), 256, 0, st>>>(p);
    }
    SRX_HIP(hipGetLastError());
    return SRX_OK;
}

int norm_run(const NormParams& p, int dtype, bool backward, hipStream_t st) {
    if (p.rows > 0) {
        const int rc = dtype == SRX_F32    ? norm_typed<float>(p, backward, st)
                       : dtype == SRX_BF16 ? norm_typed<__bf16>(p, backward, st)
                                           : norm_typed<_Float16>(p, backward, st);
        if (rc) return rc;
    }
    if (backward && (p.dweight != nullptr || p.dbias != nullptr)) {
        norm_sum_kernel<<<(unsigned)((2 * (int64_t)p.width + 31) / 32), kSumThreads, 0, st>>>(p);
        SRX_HIP(hipGetLastError());
    }
    return SRX_OK;
}

int check_norm(srx_handle_t h, int64_t rows, int32_t features, const char* who) {
    SRX_REQUIRE(h != nullptr, "%s: NULL context", who);
    SRX_REQUIRE(rows >= 0 && features >= 1, "%s: Shape mismatch (n_rows=%lld n_features=%d)", who, (long long)rows, features);
    SRX_REQUIRE(features <= kMostColumns, "%s: n_features %d above 2^24", who, features);
    return SRX_OK;
}

}  // namespace

extern "C" {

int srx_layer_norm(srx_handle_t h, const void* x, int64_t ld_x, int dtype, int64_t n_rows, int32_t n_features,
                   const float* weight, const float* bias, double eps, void* y, int64_t ld_y, float* mean,
                   float* rstd, void* stream) {
    const char* who = "srx_layer_norm";
    int rc = check_norm(h, n_rows, n_features, who);
    if (rc) return rc;
    SRX_REQUIRE(frame_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    SRX_REQUIRE(eps >= 0.0, "%s: eps must not be negative", who);
    if (n_rows == 0) return SRX_OK;
    SRX_REQUIRE(x && y && mean && rstd, "%s: NULL argument", who);
    SRX_REQUIRE(ld_x >= n_features && ld_y >= n_features, "%s: a row pitch is smaller than its row", who);
    NormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.ld_x = ld_x;
    p.rows = n_rows;
    p.width = n_features;
    p.weight = weight;
    p.bias = bias;
    p.eps = (float)eps;
    p.y = y;
    p.ld_y = ld_y;
    p.mean = mean;
    p.rstd = rstd;
    p.parts = (int64_t)h->n_cu * 8;              // workgroups that the chip holds
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return norm_run(p, dtype, false, (hipStream_t)stream);
}

int64_t srx_layer_norm_backward_workspace(srx_handle_t h, int64_t n_rows, int32_t n_features) {
    if (check_norm(h, n_rows, n_features, "srx_layer_norm_backward_workspace")) return -1;
    return norm_parts(h, n_rows, n_features) * 2 * n_features * 4;
}

int srx_layer_norm_backward(srx_handle_t h, const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int dtype,
                            int64_t n_rows, int32_t n_features, const float* mean, const float* rstd,
                            const float* weight, void* dx, int64_t ld_dx, float* dweight, float* dbias,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "srx_layer_norm_backward";
    int rc = check_norm(h, n_rows, n_features, who);
    if (rc) return rc;
    SRX_REQUIRE(frame_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    SRX_REQUIRE(n_rows == 0 || (dy && x && mean && rstd && dx), "%s: NULL argument", who);
    SRX_REQUIRE(n_rows == 0 || (ld_x >= n_features && ld_dy >= n_features && ld_dx >= n_features),
                "%s: a row pitch is smaller than its row", who);
    const int64_t need = srx_layer_norm_backward_workspace(h, n_rows, n_features);
    SRX_REQUIRE(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %lld bytes, %lld are needed", who,
                (long long)workspace_bytes, (long long)need);
    NormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.ld_x = ld_x;
    p.rows = n_rows;
    p.width = n_features;
    p.weight = weight;
    p.mean = const_cast<float*>(mean);           // (read only here)
    p.rstd = const_cast<float*>(rstd);
    p.dy = dy;
    p.ld_dy = ld_dy;
    p.dx = dx;
    p.ld_dx = ld_dx;
    p.dweight = dweight;
    p.dbias = dbias;
    p.part = (float*)workspace;
    p.parts = n_rows == 0 ? 0 : norm_parts(h, n_rows, n_features);
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return norm_run(p, dtype, true, (hipStream_t)stream);
}

}  // extern "C"
