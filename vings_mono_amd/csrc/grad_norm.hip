// Global norm of many gradient tensors, and clipping by it, on gfx950.
//
//   norm = sqrt(sum_t sum_i g_ti^2)   or   max_ti |g_ti|
//   out_ti = g_ti * min(1, max_norm / (norm + 1e-6))
//
// HBM-bound: the norm reads every gradient once, clipping reads it again and writes it.  The
// tensors travel in the kernel arguments (address, length, type), so a call copies nothing to
// the device, synchronises nothing and can be captured; a long list takes several launches.
// Every tensor is cut into chunks of 2048 elements; a workgroup owns a contiguous run of the
// chunks of all tensors, its waves take them in turn, 16 bytes per lane and load.  No atomics:
// a workgroup leaves one 64-bit partial result, and whoever needs the norm joins the partial
// results in one fixed order -- the workgroups of the scaling launch each do it for themselves
// (up to 8 KB out of the L2 for every launch that the list takes), which saves a launch between the
// two.
// Up to 16 chunks (32 K elements) one workgroup does everything in a single launch (4 us).
// Measured: norm of 144 tensors, 806 MB of bfloat16, 139 + 5 us = 5.7 TB/s; clipping 336 MB of
// bfloat16 into 671 MB of float32, 104 + 177 us (the gradients are read twice, 1.34 GB, and the norm
// launch also waits for what the caches still have to write back).  Streaming ("nontemporal") stores
// of the result took 372 us in all instead of 301, twice the workgroups 313.
//
// The reference limits gradients of its tracker network the same way between backward and the
// optimiser (scripts/frontend/modules/clipping.py); the mapping loop has no counterpart.
#include <algorithm>
#include <exception>
#include <vector>

#include "elem_types.hpp"
#include "grad_norm.hpp"

namespace vings {

constexpr int kChunk = 2048;              // elements
constexpr int kNormTensors = 160;         // per launch: 3.4 KB of kernel arguments
constexpr int kClipTensors = 112;         // ... 3.4 KB
constexpr int kFewTensors = 16;           // a list this short travels in 0.5 KB and starts sooner
                                          // (norm of 5 tensors 10.6 -> 10.3 us, clipping 19.7 -> 19.4)
constexpr int kMaxPartials = 1024;        // workgroups per launch
constexpr int kOneBlockChunks = 16;

template <int CAP, bool OUT>
struct TensorTable {
    const void* in[CAP];
    void* out[OUT ? CAP : 1];
    int64_t n[CAP];
    uint32_t first[CAP + 1];              // chunks [first[t], first[t+1]) belong to tensor t
    uint8_t type[CAP];
    uint8_t out_type[OUT ? CAP : 1];
    int count;
};

// The table as the waves read it: copied into LDS, an entry per lane.  Read where it stands, in
// the kernel arguments, every step of the search would wait for its own line out of host memory.
template <int CAP, bool OUT>
__device__ __forceinline__ void copy_table(const TensorTable<CAP, OUT>& from, TensorTable<CAP, OUT>& to) {
    for (int i = threadIdx.x; i <= from.count; i += blockDim.x) {
        to.first[i] = from.first[i];
        if (i == from.count) { to.count = from.count; break; }
        to.in[i] = from.in[i];
        to.n[i] = from.n[i];
        to.type[i] = from.type[i];
        if constexpr (OUT) { to.out[i] = from.out[i]; to.out_type[i] = from.out_type[i]; }
    }
    __syncthreads();
}

template <int CAP, bool OUT>
__device__ __forceinline__ int tensor_of(const TensorTable<CAP, OUT>& T, uint32_t chunk) {
    int lo = 0, hi = T.count - 1;         // last t with first[t] <= chunk (empty tensors are left out)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (T.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int KIND, typename T>
__device__ __forceinline__ void chunk_norm(const void* in, int64_t off, int64_t numel, double acc[4]) {
    constexpr int V = Elem<T>::kVec, R = kChunk / (64 * V);
    typedef typename Elem<T>::vec vec;
    const T* __restrict__ p = (const T*)in + off;
    const int lane = threadIdx.x & 63;
    const int64_t n = numel - off;
    if (n >= kChunk) {
        vec v[R];
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = *(const vec*)(p + (r * 64 + lane) * V);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < V; ++k) norm_take<KIND>(acc[k & 3], (float)v[r][k]);
    } else {
        // whole vectors, all in flight, then the up to V - 1 elements behind them
        const int whole = (int)n / V;
        vec v[R];
        const int at = whole * V + lane;
        const T rest = p[min(at, (int)n - 1)];
        // (unguarded: a load inside a divergent branch is waited for where the branch ends)
        if (whole > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) v[r] = *(const vec*)(p + min(r * 64 + lane, whole - 1) * V);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * 64 + lane < whole) {
#pragma unroll
                for (int k = 0; k < V; ++k) norm_take<KIND>(acc[k & 3], (float)v[r][k]);
            }
        if (at < (int)n) norm_take<KIND>(acc[0], (float)rest);
    }
}

template <int KIND, int CAP, bool OUT>
__device__ __forceinline__ double range_norm(const TensorTable<CAP, OUT>& T, uint32_t lo, uint32_t hi,
                                             int waves) {
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t c = lo + w;
    if (c < hi) {
        int t = tensor_of(T, c);
        for (; c < hi; c += waves) {
            while (c >= T.first[t + 1]) ++t;
            const int64_t off = (int64_t)(c - T.first[t]) * kChunk;
            if (T.type[t] == ELEM_F32) chunk_norm<KIND, float>(T.in[t], off, T.n[t], acc);
            else if (T.type[t] == ELEM_BF16) chunk_norm<KIND, __bf16>(T.in[t], off, T.n[t], acc);
            else chunk_norm<KIND, _Float16>(T.in[t], off, T.n[t], acc);
        }
    }
    return norm_join<KIND>(norm_join<KIND>(acc[0], acc[1]), norm_join<KIND>(acc[2], acc[3]));
}

// The wider side sets the vector: 16 bytes of it per lane, so that its accesses are contiguous
// over the lanes (16-bit gradients into float32: loads of 8 bytes).
template <typename T, typename O>
__device__ __forceinline__ void chunk_scale(const void* in, void* out, int64_t off, int64_t numel,
                                            float coef) {
    constexpr int V = Elem<O>::kVec, R = kChunk / (64 * V);
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    typedef typename Elem<O>::vec ovec;
    const T* p = (const T*)in + off;
    O* q = (O*)out + off;
    const int lane = threadIdx.x & 63;
    const int64_t n = numel - off;
    auto put = [&](int r, const vec& x) {
        ovec o;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = (O)((float)x[k] * coef);
        *(ovec*)(q + (r * 64 + lane) * V) = o;
    };
    vec v[R];
    if (n >= kChunk) {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = *(const vec*)(p + (r * 64 + lane) * V);
#pragma unroll
        for (int r = 0; r < R; ++r) put(r, v[r]);
        return;
    }
    // whole vectors, all in flight, then the up to V - 1 elements behind them
    const int whole = (int)n / V, at = whole * V + lane;
    const T rest = p[min(at, (int)n - 1)];
    if (whole > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = *(const vec*)(p + min(r * 64 + lane, whole - 1) * V);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * 64 + lane < whole) put(r, v[r]);
    if (at < (int)n) q[at] = (O)((float)rest * coef);
}

// A gradient that is already short enough stays as it is: in place, nothing is read or written.
// The chunks are taken from the last to the first: what the norm read last is still in the cache.
// (A wave's first chunk loaded ahead of the norm's join was waited for at once, the loads being in
// branches on the tensor's type, and cost 12 bytes of scratch: kernel at 300 k splats 8.8 us with it,
// 8.5 without, 5 M splats 145 and 143 us in all, 60 tensors 279 and 281.)
template <int CAP>
__device__ __forceinline__ void range_scale(const TensorTable<CAP, true>& T, uint32_t lo,
                                            uint32_t hi, int waves, float coef) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (hi <= lo + w) return;
    uint32_t c = hi - 1 - w;
    int t = tensor_of(T, c);
    for (;;) {
        while (c < T.first[t]) --t;
        if (coef != 1.0f || T.in[t] != T.out[t]) {
            const int64_t off = (int64_t)(c - T.first[t]) * kChunk;
            const int ty = T.type[t], ot = T.out_type[t];
            if (ty == ELEM_F32) chunk_scale<float, float>(T.in[t], T.out[t], off, T.n[t], coef);
            else if (ty == ELEM_BF16 && ot == ELEM_F32) chunk_scale<__bf16, float>(T.in[t], T.out[t], off, T.n[t], coef);
            else if (ty == ELEM_BF16) chunk_scale<__bf16, __bf16>(T.in[t], T.out[t], off, T.n[t], coef);
            else if (ot == ELEM_F32) chunk_scale<_Float16, float>(T.in[t], T.out[t], off, T.n[t], coef);
            else chunk_scale<_Float16, _Float16>(T.in[t], T.out[t], off, T.n[t], coef);
        }
        if (c < lo + waves) break;
        c -= waves;
    }
}

__device__ __forceinline__ void block_range(uint32_t total, uint32_t& lo, uint32_t& hi) {
    lo = (uint32_t)((uint64_t)total * blockIdx.x / gridDim.x);
    hi = (uint32_t)((uint64_t)total * (blockIdx.x + 1) / gridDim.x);
}

// One partial result per workgroup; alone, a workgroup writes the norm itself.
template <int KIND, int CAP, bool OUT>
__global__ __launch_bounds__(1024) void norm_partial_kernel(TensorTable<CAP, OUT> args,
                                                            double* __restrict__ partial,
                                                            float* __restrict__ norm) {
    __shared__ double scratch[16];
    __shared__ TensorTable<CAP, OUT> T;
    copy_table(args, T);
    uint32_t lo, hi;
    block_range(T.first[T.count], lo, hi);
    const double v = norm_join_block<KIND>(range_norm<KIND>(T, lo, hi, blockDim.x >> 6), scratch);
    if (threadIdx.x == 0) {
        if (partial) partial[blockIdx.x] = v;
        else *norm = (float)(KIND == NORM_2 ? sqrt(v) : v);
    }
}

template <int KIND>
__global__ __launch_bounds__(1024) void norm_final_kernel(const double* __restrict__ partial, int n,
                                                          float* __restrict__ norm) {
    __shared__ double scratch[16];
    const float v = norm_of_partials<KIND>(partial, n, scratch);
    if (threadIdx.x == 0) *norm = v;
}

template <int KIND, int CAP>
__global__ __launch_bounds__(256) void clip_scale_kernel(TensorTable<CAP, true> args,
                                                         const double* __restrict__ partial,
                                                         int n_partial, float max_norm,
                                                         float* __restrict__ norm) {
    __shared__ double scratch[16];
    __shared__ TensorTable<CAP, true> T;
    copy_table(args, T);
    const float v = norm_of_partials<KIND>(partial, n_partial, scratch);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
    uint32_t lo, hi;
    block_range(T.first[T.count], lo, hi);
    range_scale(T, lo, hi, 4, clip_coefficient(v, max_norm));
}

// Norm and scaling of a few chunks by one workgroup.
template <int KIND, int CAP>
__global__ __launch_bounds__(1024) void clip_one_block_kernel(TensorTable<CAP, true> args,
                                                              float max_norm,
                                                              float* __restrict__ norm) {
    __shared__ double scratch[16];
    __shared__ TensorTable<CAP, true> T;
    copy_table(args, T);
    const int waves = blockDim.x >> 6;
    const uint32_t hi = T.first[T.count];
    const double s = norm_join_block<KIND>(range_norm<KIND>(T, 0u, hi, waves), scratch);
    const float v = (float)(KIND == NORM_2 ? sqrt(s) : s);
    if (threadIdx.x == 0) *norm = v;
    range_scale(T, 0u, hi, waves, clip_coefficient(v, max_norm));
}

__global__ void norm_of_nothing_kernel(float* norm) { *norm = 0.0f; }

namespace {

inline int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// Workgroups for a launch over `chunks` chunks: a chunk per wave, at most kMaxPartials of them.
inline int blocks_for(int64_t chunks) {
    return (int)std::min<int64_t>(kMaxPartials, std::max<int64_t>(1, (chunks + 3) / 4));
}

struct ListPlan {                      // the non-empty tensors, cut into launches
    std::vector<int> index;
    std::vector<int> launch_end;       // index[launch_end[k-1] .. launch_end[k])
    std::vector<int64_t> launch_chunks;
    int64_t partials = 0, chunks = 0;
};

ListPlan plan_list(int n_tensors, const int64_t* numels, int cap) {
    ListPlan p;
    int64_t in_launch = 0;
    int held = 0;
    auto close = [&] {
        if (!held) return;
        p.launch_end.push_back((int)p.index.size());
        p.launch_chunks.push_back(in_launch);
        p.partials += blocks_for(in_launch);
        p.chunks += in_launch;
        held = 0; in_launch = 0;
    };
    for (int i = 0; i < n_tensors; ++i) {
        if (numels[i] == 0) continue;
        const int64_t c = chunks_of(numels[i]);
        if (held == cap || in_launch + c > 0xFFFFFFFFll) close();
        p.index.push_back(i);
        ++held; in_launch += c;
    }
    close();
    return p;
}

template <int CAP, bool OUT>
void fill_table(TensorTable<CAP, OUT>& T, const ListPlan& p, int launch, const void* const* in,
                void* const* out, const int64_t* n, const int* types, const int* out_types) {
    const int b = launch ? p.launch_end[launch - 1] : 0, e = p.launch_end[launch];
    T.count = e - b;
    uint32_t c = 0;
    for (int k = 0; k < T.count; ++k) {
        const int i = p.index[b + k];
        T.in[k] = in[i];
        T.n[k] = n[i];
        T.type[k] = (uint8_t)types[i];
        T.first[k] = c;
        if (OUT) { T.out[k] = out[i]; T.out_type[k] = (uint8_t)out_types[i]; }
        c += (uint32_t)chunks_of(n[i]);
    }
    T.first[T.count] = c;
}

int check_list(int n_tensors, const void* const* in, const int64_t* n, const int* types) {
    VINGS_REQUIRE(n_tensors >= 0, "sizes");
    if (n_tensors == 0) return VINGS_OK;
    VINGS_REQUIRE(in && n && types, "null pointer");
    for (int i = 0; i < n_tensors; ++i) {
        VINGS_REQUIRE(n[i] >= 0 && n[i] <= ((int64_t)1 << 42), "sizes");
        VINGS_REQUIRE(elem_known(types[i]), "element type");
        if (n[i] == 0) continue;
        VINGS_REQUIRE(in[i], "null pointer");
        VINGS_REQUIRE(((uintptr_t)in[i] & (elem_bytes(types[i]) - 1)) == 0, "element alignment");
    }
    return VINGS_OK;
}

// What is written must not lie in another tensor of the call: two waves would race.
bool writes_overlap(int n_tensors, const void* const* in, void* const* out, const int64_t* n,
                    const int* types, const int* out_types) {
    struct Span { uintptr_t b, e; int owner; bool written; };
    std::vector<Span> s;
    s.reserve(2 * (size_t)n_tensors);
    for (int i = 0; i < n_tensors; ++i) {
        if (n[i] == 0) continue;
        const uintptr_t a = (uintptr_t)in[i], o = (uintptr_t)out[i];
        const bool same = a == o && types[i] == out_types[i];
        s.push_back({o, o + (uintptr_t)n[i] * elem_bytes(out_types[i]), i, true});
        if (!same) s.push_back({a, a + (uintptr_t)n[i] * elem_bytes(types[i]), i, false});
    }
    std::sort(s.begin(), s.end(), [](const Span& x, const Span& y) { return x.b < y.b; });
    uintptr_t read_end = 0, write_end = 0;
    for (const Span& x : s) {
        if (x.b < write_end || (x.written && x.b < read_end)) return true;
        uintptr_t& end = x.written ? write_end : read_end;
        end = std::max(end, x.e);
    }
    return false;
}

template <int KIND, int CAP, bool OUT>
int launch_partials(const ListPlan& p, const void* const* in, void* const* out, const int64_t* n,
                    const int* types, const int* out_types, double* partials, hipStream_t s) {
    int64_t at = 0;
    for (int l = 0; l < (int)p.launch_end.size(); ++l) {
        TensorTable<CAP, OUT> T;
        fill_table(T, p, l, in, out, n, types, out_types);
        const int blocks = blocks_for(p.launch_chunks[l]);
        norm_partial_kernel<KIND, CAP, OUT><<<blocks, 256, 0, s>>>(T, partials + at, nullptr);
        VINGS_LAUNCH_CHECK();
        at += blocks;
    }
    return VINGS_OK;
}

template <int KIND, int CAP>
int norm_impl(int n_tensors, const void* const* in, const int64_t* n, const int* types, float* norm,
              void* workspace, hipStream_t s) {
    const ListPlan p = plan_list(n_tensors, n, CAP);
    ProfScope prof(PROF_AUX, s);
    if (p.chunks == 0) {
        norm_of_nothing_kernel<<<1, 1, 0, s>>>(norm);
        VINGS_LAUNCH_CHECK();
        return VINGS_OK;
    }
    if (p.launch_end.size() == 1 && p.chunks <= kOneBlockChunks) {
        TensorTable<CAP, false> T;
        fill_table(T, p, 0, in, nullptr, n, types, nullptr);
        norm_partial_kernel<KIND, CAP, false><<<1, 64 * (int)p.chunks, 0, s>>>(T, nullptr, norm);
        VINGS_LAUNCH_CHECK();
        return VINGS_OK;
    }
    double* partials = (double*)workspace;
    const int rc = launch_partials<KIND, CAP, false>(p, in, nullptr, n, types, nullptr, partials, s);
    if (rc != VINGS_OK) return rc;
    norm_final_kernel<KIND><<<1, 1024, 0, s>>>(partials, (int)p.partials, norm);
    VINGS_LAUNCH_CHECK();
    return VINGS_OK;
}

template <int KIND, int CAP>
int clip_impl(int n_tensors, const void* const* in, void* const* out, const int64_t* n, const int* types,
              const int* out_types, float max_norm, float* norm, void* workspace, hipStream_t s) {
    const ListPlan p = plan_list(n_tensors, n, CAP);
    ProfScope prof(PROF_AUX, s);
    if (p.chunks == 0) {
        norm_of_nothing_kernel<<<1, 1, 0, s>>>(norm);
        VINGS_LAUNCH_CHECK();
        return VINGS_OK;
    }
    if (p.launch_end.size() == 1 && p.chunks <= kOneBlockChunks) {
        TensorTable<CAP, true> T;
        fill_table(T, p, 0, in, out, n, types, out_types);
        clip_one_block_kernel<KIND, CAP><<<1, 64 * (int)p.chunks, 0, s>>>(T, max_norm, norm);
        VINGS_LAUNCH_CHECK();
        return VINGS_OK;
    }
    double* partials = (double*)workspace;
    const int rc = launch_partials<KIND, CAP, true>(p, in, out, n, types, out_types, partials, s);
    if (rc != VINGS_OK) return rc;
    for (int l = 0; l < (int)p.launch_end.size(); ++l) {
        TensorTable<CAP, true> T;
        fill_table(T, p, l, in, out, n, types, out_types);
        clip_scale_kernel<KIND, CAP><<<blocks_for(p.launch_chunks[l]), 256, 0, s>>>(
            T, partials, (int)p.partials, max_norm, l == 0 ? norm : nullptr);
        VINGS_LAUNCH_CHECK();
    }
    return VINGS_OK;
}

}  // namespace
}  // namespace vings

using namespace vings;

extern "C" size_t vings_grad_norm_workspace_bytes(int n_tensors, const int64_t* numels_host) {
    // (an upper bound for both entries: the shorter table of the clipping launches)
    if (n_tensors <= 0 || !numels_host) return 0;
    int64_t partials = 0, chunks = 0;
    int launches = 1, held = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (numels_host[i] <= 0) continue;
        const int64_t c = chunks_of(numels_host[i]);
        if (held == kClipTensors || chunks + c > 0xFFFFFFFFll) { ++launches; held = 0; chunks = 0; }
        ++held; chunks += c; partials += c / 4 + 1;
    }
    return sizeof(double) * (size_t)std::min<int64_t>(partials + launches, (int64_t)launches * kMaxPartials);
}

extern "C" int vings_grad_norm(int n_tensors, const void* const* grads_host,
                               const int64_t* numels_host, const int* types_host, int norm_kind,
                               float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    VINGS_REQUIRE(norm_kind == NORM_2 || norm_kind == NORM_MAX, "norm kind");
    VINGS_REQUIRE(norm, "null pointer");
    const int rc = check_list(n_tensors, grads_host, numels_host, types_host);
    if (rc != VINGS_OK) return rc;
    if (vings_grad_norm_workspace_bytes(n_tensors, numels_host) > workspace_bytes) {
        set_error("gradient norm workspace too small: %zu bytes", workspace_bytes);
        return VINGS_ERR_CAPACITY;
    }
    VINGS_REQUIRE(((uintptr_t)workspace & 7) == 0, "workspace must be 8-byte aligned");
    VINGS_REQUIRE(workspace || workspace_bytes == 0, "null pointer");
    try {
        const bool few = n_tensors <= kFewTensors;
        const auto impl = norm_kind == NORM_2
            ? (few ? norm_impl<NORM_2, kFewTensors> : norm_impl<NORM_2, kNormTensors>)
            : (few ? norm_impl<NORM_MAX, kFewTensors> : norm_impl<NORM_MAX, kNormTensors>);
        return impl(n_tensors, grads_host, numels_host, types_host, norm, workspace, (hipStream_t)stream);
    } catch (const std::exception& e) {
        set_error("gradient norm: %s", e.what());
        return VINGS_ERR_ARG;
    }
}

extern "C" int vings_grad_clip(int n_tensors, const void* const* grads_host, void* const* outs_host,
                               const int64_t* numels_host, const int* types_host,
                               const int* out_types_host, int norm_kind, float max_norm, float* norm,
                               void* workspace, size_t workspace_bytes, void* stream) {
    VINGS_REQUIRE(norm_kind == NORM_2 || norm_kind == NORM_MAX, "norm kind");
    VINGS_REQUIRE(max_norm >= 0.0f, "max_norm must not be negative");
    VINGS_REQUIRE(norm, "null pointer");
    const int rc = check_list(n_tensors, grads_host, numels_host, types_host);
    if (rc != VINGS_OK) return rc;
    if (n_tensors > 0) VINGS_REQUIRE(outs_host && out_types_host, "null pointer");
    for (int i = 0; i < n_tensors; ++i) {
        VINGS_REQUIRE(out_types_host[i] == types_host[i] || out_types_host[i] == ELEM_F32,
                      "a clipped gradient has its own type or float32");
        if (numels_host[i] == 0) continue;
        VINGS_REQUIRE(outs_host[i], "null pointer");
        VINGS_REQUIRE(((uintptr_t)outs_host[i] & (elem_bytes(out_types_host[i]) - 1)) == 0,
                      "element alignment");
    }
    if (vings_grad_norm_workspace_bytes(n_tensors, numels_host) > workspace_bytes) {
        set_error("gradient clip workspace too small: %zu bytes", workspace_bytes);
        return VINGS_ERR_CAPACITY;
    }
    VINGS_REQUIRE(((uintptr_t)workspace & 7) == 0, "workspace must be 8-byte aligned");
    VINGS_REQUIRE(workspace || workspace_bytes == 0, "null pointer");
    try {
        VINGS_REQUIRE(!writes_overlap(n_tensors, grads_host, outs_host, numels_host, types_host, out_types_host),
                      "a clipped gradient overlaps another tensor of the call");
        const bool few = n_tensors <= kFewTensors;
        const auto impl = norm_kind == NORM_2
            ? (few ? clip_impl<NORM_2, kFewTensors> : clip_impl<NORM_2, kClipTensors>)
            : (few ? clip_impl<NORM_MAX, kFewTensors> : clip_impl<NORM_MAX, kClipTensors>);
        return impl(n_tensors, grads_host, outs_host, numels_host, types_host, out_types_host, max_norm, norm,
                    workspace, (hipStream_t)stream);
    } catch (const std::exception& e) {
        set_error("gradient clip: %s", e.what());
        return VINGS_ERR_ARG;
    }
}
