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
template <typename I>
__device__ __forceinline__ I row_of(I e, int M) {
    switch (M) {
        case 1: return e;
        case 2: return e >> 1;
        case 3: return e / 3;
        case 4: return e >> 2;
        default: return e / (I)M;
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
// another 8 B and a launch.  HBM-bound.
// ---------------------------------------------------------------------------
constexpr int kNormBlocks = 512;       // partial results per launch
constexpr int kStepBlocks = 2048;      // eight workgroups per CU share the reading of the partials
constexpr int kMaxClipGroups = 64;

typedef Elem<float>::vec quad_t;       // 16-byte access at any 4-byte boundary

// Which of the four elements from e0 lie in visible rows (elements at or behind `total` do not).
template <typename I>
__device__ __forceinline__ int visible_quad(const uint8_t* __restrict__ visible, I e0, I total, int M) {
    if (M >= 4 && e0 + 4 <= total) {
        const I r = M == 4 ? e0 >> 2 : e0 / (I)M;
        const I left = (r + 1) * (I)M - e0;           // elements of row r from e0 on
        const int a = visible[r] ? 0xF : 0;
        if (left >= 4) return a;
        const int low = (1 << (int)left) - 1;
        return (a & low) | (visible[r + 1] ? 0xF & ~low : 0);
    }
    int m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (e0 + k < total && visible[row_of(e0 + k, M)]) m |= 1 << k;
    return m;
}

// Calls f(group, first element, length of the group's arrays, visibility bits) for every quad
// with a visible element that this workgroup serves.
template <typename F>
__device__ __forceinline__ void for_visible_quads(const AdamGroups& G, const uint8_t* __restrict__ visible,
                                                  int N, F f) {
    int g = 0;
    for (int b = blockIdx.x; b < G.first_block[G.n]; b += gridDim.x) {
        while (b >= G.first_block[g + 1]) ++g;
        const int M = G.width[g];
        const int64_t total = (int64_t)N * M;
        const int64_t e0 = ((int64_t)(b - G.first_block[g]) * 256 + threadIdx.x) * 4;
        if (e0 >= total) continue;
        // (32-bit row arithmetic wherever the array allows it: a 64-bit division is a subroutine)
        const int m = total <= 0x7FFFFFFFll ? visible_quad<uint32_t>(visible, (uint32_t)e0, (uint32_t)total, M)
                                            : visible_quad<int64_t>(visible, e0, total, M);
        if (m) f(g, e0, total, m);
    }
}

__device__ __forceinline__ void load_quad(const float* __restrict__ p, int64_t e0, int64_t total, float q[4]) {
    if (e0 + 4 <= total) {
        const quad_t v = *reinterpret_cast<const quad_t*>(p + e0);
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = e0 + k < total ? p[e0 + k] : 0.f;
    }
}

// Only a quad that is visible as a whole is stored with one access: the elements of invisible
// rows are not written, not even with their own value.
__device__ __forceinline__ void store_quad(float* __restrict__ p, int64_t e0, int m, const float q[4]) {
    if (m == 0xF) {
        quad_t v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = q[k];
        *reinterpret_cast<quad_t*>(p + e0) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((m >> k) & 1) p[e0 + k] = q[k];
    }
}

__global__ __launch_bounds__(256) void adam_norm_partial_kernel(AdamGroups G,
                                                                const uint8_t* __restrict__ visible,
                                                                int N, double* __restrict__ partial) {
    __shared__ double scratch[16];
    double acc = 0.0;
    for_visible_quads(G, visible, N, [&](int g, int64_t e0, int64_t total, int m) {
        float q[4];
        load_quad(G.grad[g], e0, total, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) norm_take<NORM_2>(acc, (m >> k) & 1 ? q[k] : 0.f);
    });
    acc = norm_join_block<NORM_2>(acc, scratch);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__global__ __launch_bounds__(256) void sparse_adam_clipped_kernel(
    AdamGroups G, const uint8_t* __restrict__ visible, float b1, float b2, float eps, int N,
    const double* __restrict__ partial, int n_partial, float max_norm, float* __restrict__ norm_out,
    const uint32_t* __restrict__ guard_count, uint32_t guard_limit) {
    __shared__ double scratch[16];
    const float norm = norm_of_partials<NORM_2>(partial, n_partial, scratch);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    if (!(norm <= 3.402823466e+38f)) return;                    // infinite or NaN: no step
    if (guard_count && *guard_count > guard_limit) return;
    const float coef = clip_coefficient(norm, max_norm);
    for_visible_quads(G, visible, N, [&](int g, int64_t e0, int64_t total, int m) {
        float p[4], d[4], mo[4], vo[4];
        load_quad(G.grad[g], e0, total, d);
        load_quad(G.param[g], e0, total, p);
        load_quad(G.m[g], e0, total, mo);
        load_quad(G.v[g], e0, total, vo);
        const float lr = G.lr[g];
#pragma unroll
        for (int k = 0; k < 4; ++k) adam_update(p[k], d[k] * coef, mo[k], vo[k], lr, b1, b2, eps);
        store_quad(G.param[g], e0, m, p);
        store_quad(G.m[g], e0, m, mo);
        store_quad(G.v[g], e0, m, vo);
    });
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
                                         const float* lrs_host, const float* b1s_host,
                                         const float* b2s_host, const float* epss_host,
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
    auto table = [&](int first, int n, AdamGroups& G) {
        int64_t blocks = 0;
        G.n = n;
        for (int k = 0; k < n; ++k) {
            const int i = first + k;
            G.param[k] = params_host[i]; G.grad[k] = grads_host[i];
            G.m[k] = exp_avgs_host[i]; G.v[k] = exp_avg_sqs_host[i];
            G.width[k] = widths_host[i]; G.lr[k] = lrs_host[i];
            G.first_block[k] = (int)blocks;
            blocks += ((int64_t)N * widths_host[i] + 1023) / 1024;
            if (blocks > 0x7FFFFFFF - kStepBlocks) return (int64_t)-1;
        }
        G.first_block[n] = (int)blocks;
        return blocks;
    };
    AdamGroups G;
    for (int i = 0; i < n_groups; i += kMaxGroups)
        VINGS_REQUIRE(table(i, std::min(kMaxGroups, n_groups - i), G) >= 0, "groups too large");
    int n_partial = 0;
    for (int i = 0; i < n_groups; i += kMaxGroups) {
        const int64_t blocks = table(i, std::min(kMaxGroups, n_groups - i), G);
        const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(kNormBlocks, blocks));
        adam_norm_partial_kernel<<<grid, 256, 0, s>>>(G, visible, N, partial + n_partial);
        VINGS_LAUNCH_CHECK();
        n_partial += grid;
    }
    for (int i = 0; i < n_groups;) {
        int n = 1;
        while (n < kMaxGroups && i + n < n_groups && b1s_host[i + n] == b1s_host[i] &&
               b2s_host[i + n] == b2s_host[i] && epss_host[i + n] == epss_host[i]) ++n;
        const int64_t blocks = table(i, n, G);
        const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(kStepBlocks, blocks));
        sparse_adam_clipped_kernel<<<grid, 256, 0, s>>>(G, visible, b1s_host[i], b2s_host[i], epss_host[i], N,
                                                        partial, n_partial, max_norm, i == 0 ? norm : nullptr,
                                                        instance_count, capacity);
        VINGS_LAUNCH_CHECK();
        i += n;
    }
    return VINGS_OK;
}
