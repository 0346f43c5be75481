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
constexpr int kNormBlocks = 1024;      // partial results per launch
constexpr int kStepBlocks = 2048;      // eight workgroups per CU share the reading of the partials
constexpr int kMaxClipGroups = 64;

typedef Elem<float>::vec quad_t;       // 16-byte access at any 4-byte boundary

// Which of the four elements from e0 (a multiple of 4) lie in visible rows; elements at or behind
// `total` do not.  Four elements touch four rows of one float, else two at most.
template <typename I>
__device__ __forceinline__ int visible_quad(const uint8_t* __restrict__ visible, I e0, I total, int M) {
    const int n = total - e0 >= 4 ? 4 : (int)(total - e0);
    if (M == 1) {
        int m = 0;
        if (n == 4) {
            typedef uint8_t u8x4 __attribute__((ext_vector_type(4), aligned(1)));
            const u8x4 v = *reinterpret_cast<const u8x4*>(visible + e0);
#pragma unroll
            for (int k = 0; k < 4; ++k) m |= v[k] ? 1 << k : 0;
        } else {
            for (int k = 0; k < n; ++k) m |= visible[e0 + k] ? 1 << k : 0;
        }
        return m;
    }
    const I r = row_of<I>(e0, M);
    const I left = (r + 1) * (I)M - e0;               // elements of row r from e0 on
    const int low = left >= 4 ? 0xF : (1 << (int)left) - 1;
    int m = visible[r] ? low : 0;
    if (left < (I)n && visible[r + 1]) m |= 0xF & ~low;
    return m & ((1 << n) - 1);
}

// A quad of one group's arrays: where it starts, and which of its elements are stepped.
struct Quad { int g, mask; int64_t e0, total; };

// The quad of this lane in block b of the launch's quads (256 consecutive ones of one group);
// mask 0 behind the end.  `g` is a hint: a group that does not lie behind b's.
__device__ __forceinline__ Quad quad_of(const AdamGroups& G, const uint8_t* __restrict__ visible, int N,
                                        int64_t b, int g) {
    Quad q{g, 0, 0, 0};
    if (b >= G.first_block[G.n]) return q;
    while (b >= G.first_block[q.g + 1]) ++q.g;
    const int M = G.width[q.g];
    q.total = (int64_t)N * M;
    q.e0 = ((b - G.first_block[q.g]) * 256 + threadIdx.x) * 4;
    if (q.e0 >= q.total) return q;
    // (32-bit row arithmetic wherever the array allows it: a 64-bit division is a subroutine)
    q.mask = q.total <= 0x7FFFFFFFll ? visible_quad<uint32_t>(visible, (uint32_t)q.e0, (uint32_t)q.total, M)
                                     : visible_quad<int64_t>(visible, q.e0, q.total, M);
    return q;
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

__device__ __forceinline__ void store_quad(float* __restrict__ p, int64_t e0, int64_t total, const float q[4]) {
    if (e0 + 4 <= total) {
        quad_t v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = q[k];
        *reinterpret_cast<quad_t*>(p + e0) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e0 + k < total) p[e0 + k] = q[k];
    }
}

// Four quads per lane and round: their visibility bytes, then their gradients are in flight
// together (one at a time the two dependent loads left this at 1 TB/s).
__global__ __launch_bounds__(256) void adam_norm_partial_kernel(AdamGroups G,
                                                                const uint8_t* __restrict__ visible,
                                                                int N, double* __restrict__ partial) {
    __shared__ double scratch[16];
    constexpr int U = 4;
    double acc[U] = {0.0, 0.0, 0.0, 0.0};
    int g = 0;
    for (int64_t b = blockIdx.x; b < G.first_block[G.n]; b += U * (int64_t)gridDim.x) {
        Quad q[U];
        float d[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = quad_of(G, visible, N, b + u * (int64_t)gridDim.x, g);
        g = q[0].g;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (q[u].mask) load_quad(G.grad[q[u].g], q[u].e0, q[u].total, d[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) norm_take<NORM_2>(acc[u], (q[u].mask >> k) & 1 ? d[u][k] : 0.f);
    }
    const double v = norm_join_block<NORM_2>((acc[0] + acc[1]) + (acc[2] + acc[3]), scratch);
    if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

struct AdamConstants { float b1, c1, b2, c2, eps; };

__global__ __launch_bounds__(256) void sparse_adam_clipped_kernel(
    AdamGroups G, const uint8_t* __restrict__ visible, AdamConstants C, int N,
    const double* __restrict__ partial, int n_partial, float max_norm, float* __restrict__ norm_out,
    const uint32_t* __restrict__ guard_count, uint32_t guard_limit) {
    __shared__ double scratch[16];
    const float norm = norm_of_partials<NORM_2>(partial, n_partial, scratch);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    if (!(norm <= 3.402823466e+38f)) return;                    // infinite or NaN: no step
    if (guard_count && *guard_count > guard_limit) return;
    const float coef = clip_coefficient(norm, max_norm);
    int g = 0;
    for (int64_t b = blockIdx.x; b < G.first_block[G.n]; b += gridDim.x) {
        const Quad q = quad_of(G, visible, N, b, g);
        g = q.g;
        if (!q.mask) continue;
        float p[4], d[4], mo[4], vo[4];
        load_quad(G.grad[g], q.e0, q.total, d);
        load_quad(G.param[g], q.e0, q.total, p);
        load_quad(G.m[g], q.e0, q.total, mo);
        load_quad(G.v[g], q.e0, q.total, vo);
        const float lr = G.lr[g];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!((q.mask >> k) & 1)) continue;       // written back as it was
            adam_update(p[k], d[k] * coef, mo[k], vo[k], lr, C.b1, C.c1, C.b2, C.c2, C.eps);
        }
        store_quad(G.param[g], q.e0, q.total, p);
        store_quad(G.m[g], q.e0, q.total, mo);
        store_quad(G.v[g], q.e0, q.total, vo);
    }
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
