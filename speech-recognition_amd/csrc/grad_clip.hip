// Gradients clipped by their global norm (srx_clip_gradients).  Two passes over the values, both memory
// bound: squares summed in 64 bits into one part per workgroup, then every workgroup adds up all parts in the
// same order (no value travels through the host, no atomics, the same bits every time) and multiplies.
// The tensors' addresses travel in the kernels' arguments, kTensors per launch, so that nothing is
// uploaded and the calls can be captured; every workgroup takes them into LDS in one go and searches there.
// 157 million bfloat16 values into float32: 296 us.  The first pass reads 3.2 TB/s (behind the writes of the call
// before), the second reads and writes 4.4 TB/s, part of its reads from the memory-side cache, which is why it runs
// backwards, in a launch and over the launches (315 us without the latter).  Stores that pass by the caches: 309 us.
#include "frame_ops.h"

#include <algorithm>
#include <vector>

using namespace srx_frames;

namespace {

constexpr int kTensors = 96;                    // 96 x 40 bytes: within the 4 KiB of a launch's arguments
constexpr int kClipThreads = 512;
constexpr int64_t kChunk = 16384;               // values that a workgroup takes at a time
constexpr int kClipVector = 8;                  // values of a thread per access

struct ClipTensor {
    void* from;
    void* to;
    int64_t count;
    int64_t chunk;                              // number of its first chunk in this launch
    int32_t dtype, to_dtype;
};
struct ClipTable {
    int32_t tensors;
    int32_t first_part, parts;                  // this launch's parts, and all launches'
    int32_t in_place;
    int64_t chunks;
    double* sums;
    double* norm;
    double max_norm;
    ClipTensor t[kTensors];
};

__device__ __forceinline__ void clip_take(const ClipTable& a, ClipTensor* table) {
    constexpr int WORDS = sizeof(ClipTensor) / 8;
    const uint64_t* from = (const uint64_t*)a.t;
    for (int i = threadIdx.x; i < a.tensors * WORDS; i += kClipThreads) ((uint64_t*)table)[i] = from[i];
    __syncthreads();
}
__device__ __forceinline__ ClipTensor clip_find(const ClipTensor* table, int tensors, int64_t chunk) {
    int lo = 0, hi = tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[mid].chunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return table[lo];
}

__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int k = 0; k < kClipThreads / 64; ++k) v += shared[k];
    return v;
}

constexpr int kClipLoads = kChunk / (kClipThreads * kClipVector);      // of a thread in a whole chunk, all in flight

// (A whole chunk and the end of a tensor part ways once, so that a whole chunk's loads are one run of instructions.)
template <typename T>
__device__ __forceinline__ double clip_squares(const T* from, int64_t count) {
    double s[2] = {0.0, 0.0};
    if (count == kChunk) {
        Pack<T, kClipVector> v[kClipLoads];
#pragma unroll
        for (int k = 0; k < kClipLoads; ++k) v[k] = load_pack<kClipVector>(from + (k * kClipThreads + (int)threadIdx.x) * kClipVector);
#pragma unroll
        for (int k = 0; k < kClipLoads; ++k)
#pragma unroll
            for (int e = 0; e < kClipVector; ++e) {
                const double d = (double)(float)v[k].v[e];
                s[e & 1] = fma(d, d, s[e & 1]);
            }
    } else {
        for (int i = threadIdx.x; i < (int)count; i += kClipThreads) {
            const double d = (double)(float)from[i];
            s[0] = fma(d, d, s[0]);
        }
    }
    return s[0] + s[1];
}

__global__ __launch_bounds__(kClipThreads) void clip_squares_kernel(ClipTable a) {
    __shared__ double shared[kClipThreads / 64];
    __shared__ ClipTensor table[kTensors];
    clip_take(a, table);
    double s = 0.0;
    for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        const ClipTensor t = clip_find(table, a.tensors, chunk);
        const int64_t at = (chunk - t.chunk) * kChunk;
        const int64_t count = min(t.count - at, kChunk);
        if (t.dtype == SRX_F32) s += clip_squares((const float*)t.from + at, count);
        else if (t.dtype == SRX_BF16) s += clip_squares((const __bf16*)t.from + at, count);
        else s += clip_squares((const _Float16*)t.from + at, count);
    }
    s = block_sum(s, shared);
    if (threadIdx.x == 0) a.sums[a.first_part + blockIdx.x] = s;
}

template <typename T, typename U>
__device__ __forceinline__ void clip_scale(const T* from, U* to, int64_t count, float factor) {
    if (count == kChunk) {
        Pack<T, kClipVector> v[kClipLoads];
#pragma unroll
        for (int k = 0; k < kClipLoads; ++k) v[k] = load_pack<kClipVector>(from + (k * kClipThreads + (int)threadIdx.x) * kClipVector);
#pragma unroll
        for (int k = 0; k < kClipLoads; ++k) {
            Pack<U, kClipVector> out;
#pragma unroll
            for (int e = 0; e < kClipVector; ++e) out.v[e] = (U)((float)v[k].v[e] * factor);
            store_pack(to + (k * kClipThreads + (int)threadIdx.x) * kClipVector, out);
        }
    } else {
        for (int i = threadIdx.x; i < (int)count; i += kClipThreads) to[i] = (U)((float)from[i] * factor);
    }
}

__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(ClipTable a) {
    __shared__ double shared[kClipThreads / 64];
    __shared__ ClipTensor table[kTensors];
    clip_take(a, table);
    double s = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += kClipThreads) s += a.sums[i];
    const double norm = sqrt(block_sum(s, shared));
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    // (a norm that is not finite says that the step is lost: the values stay as they are)
    const bool clip = norm < __builtin_huge_val() && norm + 1e-6 > a.max_norm;
    if (!clip && a.in_place) return;
    const float factor = clip ? (float)(a.max_norm / (norm + 1e-6)) : 1.0f;
    // (backwards: what the first pass read last may still lie in a cache)
    for (int64_t chunk = a.chunks - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
        const ClipTensor t = clip_find(table, a.tensors, chunk);
        const int64_t at = (chunk - t.chunk) * kChunk;
        const int64_t count = min(t.count - at, kChunk);
        if (t.dtype == SRX_F32) {
            clip_scale((const float*)t.from + at, (float*)t.to + at, count, factor);
        } else if (t.dtype == SRX_BF16) {
            if (t.to_dtype == SRX_F32) clip_scale((const __bf16*)t.from + at, (float*)t.to + at, count, factor);
            else clip_scale((const __bf16*)t.from + at, (__bf16*)t.to + at, count, factor);
        } else {
            if (t.to_dtype == SRX_F32) clip_scale((const _Float16*)t.from + at, (float*)t.to + at, count, factor);
            else clip_scale((const _Float16*)t.from + at, (_Float16*)t.to + at, count, factor);
        }
    }
}

int64_t clip_chunks(int64_t count) { return (count + kChunk - 1) / kChunk; }

// Workgroups of a launch: four per CU, or as many as there are chunks.
int64_t clip_blocks(const srx_context* h, int64_t chunks) {
    const int64_t most = (int64_t)h->n_cu * 4;
    return chunks < 1 ? 1 : chunks < most ? chunks : most;
}

// Runs `go(first, last, chunks)` for every launch's tensors.
template <typename F>
int clip_launches(int64_t n, const int64_t* counts, F go) {
    int64_t first = 0;
    do {
        int64_t last = first, chunks = 0;
        int used = 0;
        while (last < n && used < kTensors) {
            chunks += clip_chunks(counts[last]);
            used += counts[last] > 0;
            ++last;
        }
        const int rc = go(first, last, chunks);
        if (rc) return rc;
        first = last;
    } while (first < n);
    return SRX_OK;
}

int check_counts(srx_handle_t h, int64_t n, const int64_t* counts, const char* who) {
    SRX_REQUIRE(h != nullptr, "%s: NULL context", who);
    SRX_REQUIRE(n >= 0 && n <= (1 << 24), "%s: n_tensors %lld outside [0, 2^24]", who, (long long)n);
    SRX_REQUIRE(n == 0 || counts != nullptr, "%s: NULL counts", who);
    for (int64_t i = 0; i < n; ++i)
        SRX_REQUIRE(counts[i] >= 0 && counts[i] < (int64_t)1 << 48, "%s: tensor %lld has %lld values", who, (long long)i,
                    (long long)counts[i]);
    return SRX_OK;
}

size_t clip_size(int32_t dtype) { return dtype == SRX_F32 ? 4 : 2; }

struct Span {
    uintptr_t begin, end;
    bool written;
    int64_t tensor;
};

// What is written may share no byte with anything else, a tensor's own values in place excepted.
int check_overlap(std::vector<Span>& spans, bool in_place, const char* who) {
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t any_end = 0, written_end = 0;       // furthest ends so far
    for (const Span& s : spans) {
        SRX_REQUIRE(!(s.written && s.begin < any_end) && !(s.begin < written_end),
                    "%s: tensors overlap (tensor %lld%s)", who, (long long)s.tensor, in_place ? "" : " or its output");
        any_end = std::max(any_end, s.end);
        if (s.written) written_end = std::max(written_end, s.end);
    }
    return SRX_OK;
}

}  // namespace

extern "C" {

int64_t srx_clip_gradients_workspace(srx_handle_t h, int64_t n_tensors, const int64_t* counts) {
    if (check_counts(h, n_tensors, counts, "srx_clip_gradients_workspace")) return -1;
    int64_t parts = 0;
    clip_launches(n_tensors, counts, [&](int64_t, int64_t, int64_t chunks) -> int {
        parts += clip_blocks(h, chunks);
        return SRX_OK;
    });
    return parts * (int64_t)sizeof(double);
}

int srx_clip_gradients(srx_handle_t h, int64_t n_tensors, void* const* tensors, const int64_t* counts,
                       const int32_t* dtypes, void* const* outs, const int32_t* out_dtypes, double max_norm,
                       double* out_norm, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "srx_clip_gradients";
    int rc = check_counts(h, n_tensors, counts, who);
    if (rc) return rc;
    SRX_REQUIRE(n_tensors == 0 || (tensors != nullptr && dtypes != nullptr), "%s: NULL tensors or dtypes", who);
    SRX_REQUIRE(outs == nullptr || n_tensors == 0 || out_dtypes != nullptr, "%s: NULL out_dtypes", who);
    SRX_REQUIRE(out_norm != nullptr, "%s: NULL out_norm", who);
    SRX_REQUIRE(max_norm >= 0.0, "%s: max_norm must not be negative", who);
    try {
        std::vector<Span> spans;
        spans.reserve((size_t)n_tensors * (outs != nullptr ? 2 : 1));
        for (int64_t i = 0; i < n_tensors; ++i) {
            SRX_REQUIRE(frame_dtype(dtypes[i]), "%s: unknown dtype %d", who, dtypes[i]);
            SRX_REQUIRE(outs == nullptr || out_dtypes[i] == dtypes[i] || out_dtypes[i] == SRX_F32,
                        "%s: output %lld must have its tensor's type or float32", who, (long long)i);
            if (counts[i] == 0) continue;
            SRX_REQUIRE(tensors[i] != nullptr && (outs == nullptr || outs[i] != nullptr), "%s: tensor %lld is NULL", who,
                        (long long)i);
            const uintptr_t at = (uintptr_t)tensors[i];
            spans.push_back({at, at + counts[i] * clip_size(dtypes[i]), outs == nullptr, i});
            if (outs != nullptr) {
                const uintptr_t to = (uintptr_t)outs[i];
                spans.push_back({to, to + counts[i] * clip_size(out_dtypes[i]), true, i});
            }
        }
        if ((rc = check_overlap(spans, outs == nullptr, who))) return rc;
    } catch (const std::bad_alloc&) {
        srx_set_error("%s: out of host memory", who);
        return SRX_ENOMEM;
    }
    const int64_t need = srx_clip_gradients_workspace(h, n_tensors, counts);
    SRX_REQUIRE(workspace != nullptr && workspace_bytes >= need, "%s: workspace of %lld bytes, %lld are needed", who,
                (long long)workspace_bytes, (long long)need);
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    hipStream_t st = (hipStream_t)stream;
    struct Launch {
        int64_t first, last, chunks, part;
    };
    std::vector<Launch> launches;
    try {
        launches.reserve((size_t)(n_tensors / kTensors + 1));
        int64_t part = 0;
        clip_launches(n_tensors, counts, [&](int64_t first, int64_t last, int64_t chunks) -> int {
            launches.push_back({first, last, chunks, part});
            part += clip_blocks(h, chunks);
            return SRX_OK;
        });
    } catch (const std::bad_alloc&) {
        srx_set_error("%s: out of host memory", who);
        return SRX_ENOMEM;
    }
    for (int pass = 0; pass < 2; ++pass) {
        for (const Launch& l : launches) {
            ClipTable a;
            a.tensors = 0;
            a.first_part = (int32_t)l.part;
            a.parts = (int32_t)(need / (int64_t)sizeof(double));
            a.in_place = outs == nullptr;
            a.chunks = l.chunks;
            a.sums = (double*)workspace;
            a.norm = out_norm;
            a.max_norm = max_norm;
            int64_t at = 0;
            for (int64_t i = l.first; i < l.last; ++i) {
                if (counts[i] == 0) continue;
                ClipTensor& t = a.t[a.tensors++];
                t.from = tensors[i];
                t.to = outs != nullptr ? outs[i] : tensors[i];
                t.count = counts[i];
                t.chunk = at;
                t.dtype = dtypes[i];
                t.to_dtype = outs != nullptr ? out_dtypes[i] : dtypes[i];
                at += clip_chunks(counts[i]);
            }
            const int64_t blocks = clip_blocks(h, l.chunks);
            if (pass == 0) clip_squares_kernel<<<(unsigned)blocks, kClipThreads, 0, st>>>(a);
            else clip_scale_kernel<<<(unsigned)blocks, kClipThreads, 0, st>>>(a);
            SRX_HIP(hipGetLastError());
        }
        std::reverse(launches.begin(), launches.end());      // (the second pass begins where the first has ended)
    }
    return SRX_OK;
}

}  // extern "C"
