// Row-masked Adam for splat parameters on gfx950 (HBM-bound elementwise op).
//
// Rows whose visibility flag is 0 keep their values: their moments do not decay.
// No bias correction, no weight decay.
// Serves SparseGaussianAdam.step as called at
// /root/reference/scripts/gaussian/gaussian_base.py:62,402 and
// /root/reference/scripts/gaussian/sky_utils.py:181.
#include <algorithm>

#include "elem_types.hpp"
#include "grad_norm.hpp"

namespace vings {

__global__ __launch_bounds__(256) void sparse_adam_kernel(
    float* __restrict__ param, const float* __restrict__ grad, float* __restrict__ exp_avg,
    float* __restrict__ exp_avg_sq, const uint8_t* __restrict__ visible, float lr, float b1,
    float b2, float eps, int64_t total, int M) {
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        if (!visible[i / M]) continue;
        float p = param[i], m = exp_avg[i], v = exp_avg_sq[i];
        adam_update(p, grad[i], m, v, lr, b1, b2, eps);
        param[i] = p; exp_avg[i] = m; exp_avg_sq[i] = v;
    }
}

constexpr int kMaxGroups = 8;
struct AdamGroups {
    float* param[kMaxGroups];
    const float* grad[kMaxGroups];
    float* m[kMaxGroups];
    float* v[kMaxGroups];
    int width[kMaxGroups];
    float lr[kMaxGroups];
    int first_block[kMaxGroups + 1];   // blocks [first_block[g], first_block[g+1]) serve group g
    int n;
};

// Row of element e in an array of rows of M floats; the widths that occur are constants.
__device__ __forceinline__ int64_t row_of(int64_t e, int M) {
    switch (M) {
        case 1: return e;
        case 2: return e >> 1;
        case 3: return e / 3;
        case 4: return e >> 2;
        default: return e / M;
    }
}

// All groups in one launch, element-parallel: a lane owns four consecutive floats of one
// group's arrays (one 16-byte load / store per array: fully coalesced, where a lane per row
// would walk rows of 4 to 16 bytes with strided scalar accesses).  A quad none of whose rows
// is visible is not touched at all; in a quad that straddles a visible and an invisible row
// the invisible elements are written back unchanged.
__global__ __launch_bounds__(256) void sparse_adam_multi_kernel(AdamGroups G,
                                                                const uint8_t* __restrict__ visible,
                                                                float b1, float b2, float eps,
                                                                int N,
                                                                const uint32_t* __restrict__ guard_count,
                                                                uint32_t guard_limit) {
    // (see vings_sparse_adam_multi_guarded: a step whose gradients are incomplete is skipped)
    if (guard_count && *guard_count > guard_limit) return;
    int g = 0;
    while (g + 1 < G.n && (int)blockIdx.x >= G.first_block[g + 1]) ++g;
    const int M = G.width[g];
    const float lr = G.lr[g];
    const int64_t total = (int64_t)N * M;
    const int64_t e0 = ((int64_t)(blockIdx.x - G.first_block[g]) * 256 + threadIdx.x) * 4;
    if (e0 >= total) return;
    float* __restrict__ P = G.param[g];
    const float* __restrict__ Gr = G.grad[g];
    float* __restrict__ Mo = G.m[g];
    float* __restrict__ Vo = G.v[g];
    if (e0 + 4 <= total) {
        bool vis[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) vis[k] = visible[row_of(e0 + k, M)] != 0;
        if (!(vis[0] | vis[1] | vis[2] | vis[3])) return;
        float4 p4 = *reinterpret_cast<float4*>(P + e0);
        const float4 g4 = *reinterpret_cast<const float4*>(Gr + e0);
        float4 m4 = *reinterpret_cast<float4*>(Mo + e0);
        float4 v4 = *reinterpret_cast<float4*>(Vo + e0);
        if (vis[0]) adam_update(p4.x, g4.x, m4.x, v4.x, lr, b1, b2, eps);
        if (vis[1]) adam_update(p4.y, g4.y, m4.y, v4.y, lr, b1, b2, eps);
        if (vis[2]) adam_update(p4.z, g4.z, m4.z, v4.z, lr, b1, b2, eps);
        if (vis[3]) adam_update(p4.w, g4.w, m4.w, v4.w, lr, b1, b2, eps);
        *reinterpret_cast<float4*>(P + e0) = p4;
        *reinterpret_cast<float4*>(Mo + e0) = m4;
        *reinterpret_cast<float4*>(Vo + e0) = v4;
    } else {
        for (int64_t e = e0; e < total; ++e) {
            if (!visible[row_of(e, M)]) continue;
            float p = P[e], m = Mo[e], v = Vo[e];
            adam_update(p, Gr[e], m, v, lr, b1, b2, eps);
            P[e] = p; Mo[e] = m; Vo[e] = v;
        }
    }
}

// ---------------------------------------------------------------------------
// The same step on gradients clipped by their global norm over the rows it applies:
//   norm = sqrt(sum over groups and visible rows of g^2),  g' = g * min(1, max_norm / (norm + 1e-6))
// Two launches: partial sums (64-bit, one per workgroup), then the update, whose workgroups
// join the partial sums themselves.  The clipped gradients are never written: per visible
// element 4 B of gradient twice and 24 B of parameter and moments, where clipping first moves
// another 8 B and a launch.  HBM-bound: 1 M splats with 0.7 of them visible at random (so that
// nearly every 64-byte line holds a visible row and 364 MB move) take 18 + 68 us, the update at
// 5.3 TB/s; the norm launch waits on its own loads and on the write-back of the step before.
// ---------------------------------------------------------------------------
constexpr int kNormBlocks = 1024;      // partial results per launch
constexpr int kStepBlocks = 2048;      // eight workgroups per CU share the reading of the partials
constexpr int kMaxClipGroups = 64;
constexpr int kNormQuads = 4;          // quads per lane and round of either launch: what is in
constexpr int kStepQuads = 2;          // flight together

typedef Elem<float>::vec quad_t;       // 16-byte access at any 4-byte boundary

// Which of the four elements from e0 (a multiple of 4, e0 + 4 <= N * width) lie in visible rows of
// W floats (W = 0: of `width` >= 2 floats).  Four elements touch four rows of one float, else two at
// most; the loads are not guarded (see below), the second row is clamped instead.
template <int W, typename I>
__device__ __forceinline__ int visible_quad(const uint8_t* __restrict__ visible, I e0, int N, int width) {
    if (W == 1) {
        typedef uint32_t u32u __attribute__((aligned(1)));
        const uint32_t v = *reinterpret_cast<const u32u*>(visible + e0);
        return (v & 0xFFu ? 1 : 0) | (v & 0xFF00u ? 2 : 0) | (v & 0xFF0000u ? 4 : 0) | (v >> 24 ? 8 : 0);
    }
    const I M = W ? (I)W : (I)width;
    const I r = e0 / M;
    if (W == 4) return visible[r] ? 0xF : 0;
    const I left = (r + 1) * M - e0;                  // elements of row r from e0 on
    const int low = left >= 4 ? 0xF : (1 << (int)left) - 1;
    const uint8_t a = visible[r], b = visible[r + 1 < (I)N ? r + 1 : r];
    return (a ? low : 0) | (b ? 0xF & ~low : 0);
}

// What a launch does with the arrays of one group: block<W, I>(group, first quad, quads) serves
// 256 * quads-per-lane quads of four elements, tail(group, e0, n) the up to three elements behind
// the last whole quad, one lane each.
//
// All loads of a block are issued for every lane, lanes behind the end taking the last quad again:
// a load inside a divergent branch is waited for where the branch ends, and a lane's loads then
// follow one another instead of being in flight together (norm launch at 1 M splats: 27 -> 18 us).
// The row widths of a splat map are constants, and indexes have 32 bits wherever the arrays
// allow it (a 64-bit division is a subroutine).
template <typename F>
__device__ __forceinline__ void for_blocks(const AdamGroups& G, int N, int per_lane, F f) {
    int g = 0;
    for (int64_t b = blockIdx.x; b < G.first_block[G.n]; b += gridDim.x) {
        while (b >= G.first_block[g + 1]) ++g;
        const int64_t total = (int64_t)N * G.width[g], quads = total >> 2;
        const int64_t first = (b - G.first_block[g]) * 256 * per_lane;
        if (first < quads) {
            if (total > 0x7FFFFFFFll - 8192) {
                if (G.width[g] == 1) f.template block<1, int64_t>(g, first, quads);
                else f.template block<0, int64_t>(g, first, quads);
            } else {
                const uint32_t f32 = (uint32_t)first, q32 = (uint32_t)quads;
                switch (G.width[g]) {
                    case 1: f.template block<1, uint32_t>(g, f32, q32); break;
                    case 2: f.template block<2, uint32_t>(g, f32, q32); break;
                    case 3: f.template block<3, uint32_t>(g, f32, q32); break;
                    case 4: f.template block<4, uint32_t>(g, f32, q32); break;
                    default: f.template block<0, uint32_t>(g, f32, q32); break;
                }
            }
        }
        // (the last block of a group; it exists for the tail alone where total < 4)
        if ((total & 3) && first + 256 * per_lane > quads && (int)threadIdx.x < (int)(total & 3))
            f.tail(g, quads * 4 + threadIdx.x);
    }
}

struct SquareSum {
    const AdamGroups& G;
    const uint8_t* __restrict__ visible;
    int N;
    double (&acc)[kNormQuads];

    template <int W, typename I>
    __device__ __forceinline__ void block(int g, I first, I quads) {
        int mask[kNormQuads];
        quad_t d[kNormQuads];
        const float* __restrict__ grad = G.grad[g];
#pragma unroll
        for (int u = 0; u < kNormQuads; ++u) {
            const I q = first + u * 256 + threadIdx.x, e0 = (q < quads ? q : quads - 1) * 4;
            d[u] = *reinterpret_cast<const quad_t*>(grad + e0);
            mask[u] = visible_quad<W, I>(visible, e0, N, G.width[g]);
        }
#pragma unroll
        for (int u = 0; u < kNormQuads; ++u) {
            const int m = first + u * 256 + threadIdx.x < quads ? mask[u] : 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) norm_take<NORM_2>(acc[u], (m >> k) & 1 ? d[u][k] : 0.f);
        }
    }
    __device__ __forceinline__ void tail(int g, int64_t e) {
        if (visible[e / G.width[g]]) norm_take<NORM_2>(acc[0], G.grad[g][e]);
    }
};

__global__ __launch_bounds__(256) void adam_norm_partial_kernel(AdamGroups G,
                                                                const uint8_t* __restrict__ visible,
                                                                int N, double* __restrict__ partial) {
    __shared__ double scratch[16];
    double acc[kNormQuads] = {};
    for_blocks(G, N, kNormQuads, SquareSum{G, visible, N, acc});
    const double v = norm_join_block<NORM_2>((acc[0] + acc[1]) + (acc[2] + acc[3]), scratch);
    if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

struct AdamConstants { float b1, c1, b2, c2, eps; };

struct ClippedUpdate {
    const AdamGroups& G;
    const uint8_t* __restrict__ visible;
    int N;
    AdamConstants C;
    float coef;

    template <int W, typename I>
    __device__ __forceinline__ void block(int g, I first, I quads) {
        int mask[kStepQuads], any = 0;
        quad_t p[kStepQuads], d[kStepQuads], m[kStepQuads], v[kStepQuads];
        I e0[kStepQuads];
#pragma unroll
        for (int u = 0; u < kStepQuads; ++u) {
            const I q = first + u * 256 + threadIdx.x;
            e0[u] = (q < quads ? q : quads - 1) * 4;
            mask[u] = visible_quad<W, I>(visible, e0[u], N, G.width[g]);
        }
#pragma unroll
        for (int u = 0; u < kStepQuads; ++u) {
            if (first + u * 256 + threadIdx.x >= quads) mask[u] = 0;
            any |= mask[u];
        }
        if (__ballot(any) == 0) return;               // nothing of this wave's quads is stepped
#pragma unroll
        for (int u = 0; u < kStepQuads; ++u) {
            d[u] = *reinterpret_cast<const quad_t*>(G.grad[g] + e0[u]);
            p[u] = *reinterpret_cast<const quad_t*>(G.param[g] + e0[u]);
            m[u] = *reinterpret_cast<const quad_t*>(G.m[g] + e0[u]);
            v[u] = *reinterpret_cast<const quad_t*>(G.v[g] + e0[u]);
        }
        const float lr = G.lr[g];
#pragma unroll
        for (int u = 0; u < kStepQuads; ++u) {
            if (!mask[u]) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float pk = p[u][k], mk = m[u][k], vk = v[u][k];
                adam_update(pk, d[u][k] * coef, mk, vk, lr, C.b1, C.c1, C.b2, C.c2, C.eps);
                const bool step = (mask[u] >> k) & 1;  // else written back as it was
                p[u][k] = step ? pk : p[u][k];
                m[u][k] = step ? mk : m[u][k];
                v[u][k] = step ? vk : v[u][k];
            }
            *reinterpret_cast<quad_t*>(G.param[g] + e0[u]) = p[u];
            *reinterpret_cast<quad_t*>(G.m[g] + e0[u]) = m[u];
            *reinterpret_cast<quad_t*>(G.v[g] + e0[u]) = v[u];
        }
    }
    __device__ __forceinline__ void tail(int g, int64_t e) {
        if (!visible[e / G.width[g]]) return;
        float p = G.param[g][e], m = G.m[g][e], v = G.v[g][e];
        adam_update(p, G.grad[g][e] * coef, m, v, G.lr[g], C.b1, C.c1, C.b2, C.c2, C.eps);
        G.param[g][e] = p; G.m[g][e] = m; G.v[g][e] = v;
    }
};

__global__ __launch_bounds__(256) void sparse_adam_clipped_kernel(
    AdamGroups G, const uint8_t* __restrict__ visible, AdamConstants C, int N,
    const double* __restrict__ partial, int n_partial, float max_norm, float* __restrict__ norm_out,
    const uint32_t* __restrict__ guard_count, uint32_t guard_limit) {
    __shared__ double scratch[16];
    // (a dropped step's gradients are incomplete, or those of the step before: it has no norm)
    const bool dropped = guard_count && *guard_count > guard_limit;
    const float norm = dropped ? __builtin_inff() : norm_of_partials<NORM_2>(partial, n_partial, scratch);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    if (!(norm <= 3.402823466e+38f)) return;                    // infinite or NaN: no step
    for_blocks(G, N, kStepQuads, ClippedUpdate{G, visible, N, C, clip_coefficient(norm, max_norm)});
}

}  // namespace vings

using namespace vings;

extern "C" int vings_sparse_adam(float* param, const float* grad, float* exp_avg,
                                 float* exp_avg_sq, const uint8_t* visible, float lr, float b1,
                                 float b2, float eps, int N, int M, void* stream) {
    VINGS_REQUIRE(N >= 0 && M > 0, "sizes");
    if (N == 0) return VINGS_OK;
    VINGS_REQUIRE(param && grad && exp_avg && exp_avg_sq && visible, "null pointer");
    const int64_t total = (int64_t)N * M;
    int blocks = cdiv(total, 256);
    if (blocks > 2048) blocks = 2048;
    ProfScope prof(PROF_ADAM, (hipStream_t)stream);
    sparse_adam_kernel<<<blocks, 256, 0, (hipStream_t)stream>>>(param, grad, exp_avg, exp_avg_sq,
                                                                visible, lr, b1, b2, eps, total, M);
    VINGS_LAUNCH_CHECK();
    return VINGS_OK;
}

static int adam_multi(int n_groups, float* const* params_host, const float* const* grads_host,
                      float* const* exp_avgs_host, float* const* exp_avg_sqs_host,
                      const int* widths_host, const float* lrs_host, const uint8_t* visible,
                      float b1, float b2, float eps, int N, void* stream,
                      const uint32_t* guard_count, uint32_t guard_limit) {
    VINGS_REQUIRE(n_groups > 0 && n_groups <= kMaxGroups, "1..8 groups");
    VINGS_REQUIRE(N >= 0, "sizes");
    if (N == 0) return VINGS_OK;
    VINGS_REQUIRE(params_host && grads_host && exp_avgs_host && exp_avg_sqs_host && widths_host &&
                      lrs_host && visible,
                  "null pointer");
    AdamGroups G;
    G.n = n_groups;
    for (int i = 0; i < n_groups; ++i) {
        VINGS_REQUIRE(params_host[i] && grads_host[i] && exp_avgs_host[i] && exp_avg_sqs_host[i] &&
                          widths_host[i] > 0,
                      "group pointers");
        G.param[i] = params_host[i];
        G.grad[i] = grads_host[i];
        G.m[i] = exp_avgs_host[i];
        G.v[i] = exp_avg_sqs_host[i];
        G.width[i] = widths_host[i];
        G.lr[i] = lrs_host[i];
    }
    int blocks = 0;
    for (int i = 0; i < n_groups; ++i) {
        VINGS_REQUIRE((((uintptr_t)G.param[i] | (uintptr_t)G.grad[i] | (uintptr_t)G.m[i] |
                        (uintptr_t)G.v[i]) & 15) == 0, "group arrays must be 16-byte aligned");
        G.first_block[i] = blocks;
        blocks += cdiv((int64_t)N * G.width[i], 1024);
    }
    G.first_block[n_groups] = blocks;
    ProfScope prof(PROF_ADAM, (hipStream_t)stream);
    sparse_adam_multi_kernel<<<blocks, 256, 0, (hipStream_t)stream>>>(G, visible, b1, b2, eps, N,
                                                                      guard_count, guard_limit);
    VINGS_LAUNCH_CHECK();
    return VINGS_OK;
}

extern "C" int vings_sparse_adam_multi(int n_groups, float* const* params_host,
                                       const float* const* grads_host,
                                       float* const* exp_avgs_host,
                                       float* const* exp_avg_sqs_host, const int* widths_host,
                                       const float* lrs_host, const uint8_t* visible, float b1,
                                       float b2, float eps, int N, void* stream) {
    return adam_multi(n_groups, params_host, grads_host, exp_avgs_host, exp_avg_sqs_host,
                      widths_host, lrs_host, visible, b1, b2, eps, N, stream, nullptr, 0u);
}

extern "C" int vings_sparse_adam_multi_guarded(int n_groups, float* const* params_host,
                                               const float* const* grads_host,
                                               float* const* exp_avgs_host,
                                               float* const* exp_avg_sqs_host,
                                               const int* widths_host, const float* lrs_host,
                                               const uint8_t* visible, float b1, float b2,
                                               float eps, int N, const uint32_t* instance_count,
                                               uint32_t capacity, void* stream) {
    VINGS_REQUIRE(instance_count != nullptr, "instance_count");
    return adam_multi(n_groups, params_host, grads_host, exp_avgs_host, exp_avg_sqs_host,
                      widths_host, lrs_host, visible, b1, b2, eps, N, stream, instance_count,
                      capacity);
}

extern "C" size_t vings_sparse_adam_clipped_workspace_bytes(int n_groups) {
    return n_groups > 0 ? sizeof(double) * kNormBlocks * (size_t)cdiv(n_groups, kMaxGroups) : 0;
}

extern "C" int vings_sparse_adam_clipped(int n_groups, float* const* params_host,
                                         const float* const* grads_host, float* const* exp_avgs_host,
                                         float* const* exp_avg_sqs_host, const int* widths_host,
                                         const float* lrs_host, const double* b1s_host,
                                         const double* b2s_host, const float* epss_host,
                                         const uint8_t* visible, int N, float max_norm, float* norm,
                                         void* workspace, size_t workspace_bytes,
                                         const uint32_t* instance_count, uint32_t capacity,
                                         void* stream) {
    VINGS_REQUIRE(n_groups > 0 && n_groups <= kMaxClipGroups, "1..64 groups");
    VINGS_REQUIRE(N >= 0, "sizes");
    VINGS_REQUIRE(max_norm >= 0.0f, "max_norm must not be negative");
    VINGS_REQUIRE(norm && workspace, "null pointer");
    VINGS_REQUIRE(((uintptr_t)workspace & 7) == 0, "workspace must be 8-byte aligned");
    if (workspace_bytes < vings_sparse_adam_clipped_workspace_bytes(n_groups)) {
        set_error("clipped Adam workspace too small: %zu bytes", workspace_bytes);
        return VINGS_ERR_CAPACITY;
    }
    VINGS_REQUIRE(params_host && grads_host && exp_avgs_host && exp_avg_sqs_host && widths_host &&
                      lrs_host && b1s_host && b2s_host && epss_host && (visible || N == 0),
                  "null pointer");
    for (int i = 0; i < n_groups; ++i) {
        VINGS_REQUIRE(widths_host[i] > 0, "group widths");
        VINGS_REQUIRE(N == 0 || (params_host[i] && grads_host[i] && exp_avgs_host[i] && exp_avg_sqs_host[i]),
                      "group pointers");
        VINGS_REQUIRE((((uintptr_t)params_host[i] | (uintptr_t)grads_host[i] | (uintptr_t)exp_avgs_host[i] |
                        (uintptr_t)exp_avg_sqs_host[i]) & 3) == 0, "group arrays must be 4-byte aligned");
    }
    hipStream_t s = (hipStream_t)stream;
    ProfScope prof(PROF_ADAM, s);
    double* partial = (double*)workspace;
    // one run of up to 8 consecutive groups per launch; an update launch also ends where the
    // next group has other constants
    auto table = [&](int first, int n, int quads, AdamGroups& G) {
        int64_t blocks = 0;
        G.n = n;
        for (int k = 0; k < n; ++k) {
            const int i = first + k;
            G.param[k] = params_host[i]; G.grad[k] = grads_host[i];
            G.m[k] = exp_avgs_host[i]; G.v[k] = exp_avg_sqs_host[i];
            G.width[k] = widths_host[i]; G.lr[k] = lrs_host[i];
            G.first_block[k] = (int)blocks;
            blocks += ((int64_t)N * widths_host[i] + 1024 * quads - 1) / (1024 * quads);
            if (blocks > 0x7FFFFFFF) return (int64_t)-1;
        }
        G.first_block[n] = (int)blocks;
        return blocks;
    };
    AdamGroups G;
    for (int i = 0; i < n_groups; i += kMaxGroups)
        VINGS_REQUIRE(table(i, std::min(kMaxGroups, n_groups - i), kStepQuads, G) >= 0, "groups too large");
    int n_partial = 0;
    for (int i = 0; i < n_groups; i += kMaxGroups) {
        const int64_t blocks = table(i, std::min(kMaxGroups, n_groups - i), kNormQuads, G);
        const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(kNormBlocks, blocks));
        adam_norm_partial_kernel<<<grid, 256, 0, s>>>(G, visible, N, partial + n_partial);
        VINGS_LAUNCH_CHECK();
        n_partial += grid;
    }
    for (int i = 0; i < n_groups;) {
        int n = 1;
        while (n < kMaxGroups && i + n < n_groups && b1s_host[i + n] == b1s_host[i] &&
               b2s_host[i + n] == b2s_host[i] && epss_host[i + n] == epss_host[i]) ++n;
        const int64_t blocks = table(i, n, kStepQuads, G);
        const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(kStepBlocks, blocks));
        // 1 - beta is formed in 64 bits: float32(1) - float32(0.999) is 1.3e-5 off
        const AdamConstants C{(float)b1s_host[i], (float)(1.0 - b1s_host[i]), (float)b2s_host[i],
                              (float)(1.0 - b2s_host[i]), epss_host[i]};
        sparse_adam_clipped_kernel<<<grid, 256, 0, s>>>(G, visible, C, N, partial, n_partial, max_norm,
                                                        i == 0 ? norm : nullptr, instance_count, capacity);
        VINGS_LAUNCH_CHECK();
        i += n;
    }
    return VINGS_OK;
}
