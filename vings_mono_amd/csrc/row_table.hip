// Rows of a table by integer id, scaled, and the gradient of that table, on gfx950.
//
//   lookup     out[n] = scale * table[id[n]]                     (zeros where id[n] names no row)
//   gradient   dtable[v] = scale * sum over {n : id[n] = v} of g[n],   touched[v] = any such n
//
// Both are HBM-bound.  The lookup is one gather: a wave takes a row (or several short ones, a
// lane group each) with 16-byte accesses, four in flight per lane.
//
// The gradient sums by SORTED ids, with no float atomics, so its bits do not depend on timing:
//   1. the ids and their positions are ordered by a stable radix sort; ids that name no row sort
//      behind the last row.  Up to 16384 ids one workgroup sorts them in LDS (registers hold the
//      pairs between the passes) while the other workgroups of the launch clear dtable and
//      touched, which takes longer than the sort when the table is large; more ids take the
//      tile passes of radix_sort.hpp, 8 bits each, of which a table of 255 rows needs one
//   2. segment kernel: the sorted positions are cut into pieces of equal length, whatever rows
//      they belong to, so one frequent id costs no more than many rare ones.  A lane group walks
//      a few consecutive positions, holds its columns' sum in float32 registers, and writes a
//      row whenever a run of equal ids begins and ends inside its piece
//   3. runs that cross lane groups are joined in LDS by a segmented scan over the groups (in
//      sorted order the run of group g continues that of group g - s exactly if their last and
//      first ids are equal), runs that cross workgroups leave one partial row per workgroup
//   4. join kernel: the workgroup in whose piece such a run begins adds the partial rows of the
//      pieces behind it, in a fixed tree
// Sums are float32 over at most 64 terms in a row, then trees; the result is scaled and rounded
// to the gradient's type once.
//
// Serves per-keyframe rows that every splat reads through the keyframe that owns it
// (globalkf_id, /root/reference/scripts/gaussian/gaussian_model.py:163-168) and any wide table;
// the reference itself has no learned table.
#include <algorithm>

#include "elem_types.hpp"
#include "radix_sort.hpp"

namespace vings {

constexpr int kLdsSortMax = 16384;        // ids one workgroup sorts
constexpr int kPieceMax = 2048;           // sorted positions per workgroup of the segment kernel

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
// Column of a lane's vector: the last one is moved back so that it ends with the row (its
// columns are then computed by two lanes, which store the same bits); V = 1 needs no moving.
template <int V>
__device__ __forceinline__ int64_t vec_col(int64_t j, int64_t D) {
    const int64_t c = j * V;
    return c + V <= D ? c : D - V;
}

template <typename T, int V> struct VecOf { typedef typename Elem<T>::vec type; };
template <typename T> struct VecOf<T, 1> { typedef T type; };

template <typename T, int V>
__device__ __forceinline__ void unpack(const typename VecOf<T, V>::type& v, float f[V]) {
    if constexpr (V == 1) f[0] = (float)v;
    else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = (float)v[k];
    }
}

template <typename O, int V>
__device__ __forceinline__ void store_cols(O* __restrict__ p, const float f[V]) {
    if constexpr (V == 1) *p = (O)f[0];
    else if constexpr (V == Elem<O>::kVec) {
        typename Elem<O>::vec o;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = (O)f[k];
        *reinterpret_cast<typename Elem<O>::vec*>(p) = o;
    } else {                               // eight 16-bit inputs to float32: two vectors
        static_assert(V == 8 && Elem<O>::kVec == 4, "");
        store_cols<O, 4>(p, f);
        store_cols<O, 4>(p + 4, f + 4);
    }
}

// A row per lane group of 2^LG lanes, four rows at a time; rows of up to 64 vectors.
template <typename T, typename I, int V>
__global__ __launch_bounds__(256) void row_lookup_kernel(
    int64_t N, int64_t D, const T* __restrict__ table, int64_t ld, const I* __restrict__ ids,
    IdRange range, float scale, T* __restrict__ out, int lg) {
    typedef typename VecOf<T, V>::type vec;
    const int64_t groups = (int64_t)gridDim.x * (256 >> lg);
    const int64_t g = (int64_t)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
    const int j = threadIdx.x & ((1 << lg) - 1);
    if ((int64_t)j * V >= D) return;
    const int64_t c = vec_col<V>(j, D);
    for (int64_t n0 = g; n0 < N; n0 += 4 * groups) {
        uint32_t row[4];
        vec v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t n = n0 + u * groups;
            row[u] = n < N ? sort_key(ids[n], range) : range.rows;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (row[u] < range.rows) v[u] = *reinterpret_cast<const vec*>(table + (int64_t)row[u] * ld + c);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t n = n0 + u * groups;
            if (n >= N) break;
            float f[V];
            unpack<T, V>(v[u], f);
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = row[u] < range.rows ? f[k] * scale : 0.f;
            store_cols<T, V>(out + n * D + c, f);
        }
    }
}

// Rows of more than 64 vectors: a wave per (row, 256 vectors of it), four vectors per lane.
template <typename T, typename I>
__global__ __launch_bounds__(256) void row_lookup_wide_kernel(
    int64_t N, int64_t D, int segments, const T* __restrict__ table, int64_t ld,
    const I* __restrict__ ids, IdRange range, float scale, T* __restrict__ out) {
    constexpr int V = Elem<T>::kVec;
    typedef typename Elem<T>::vec vec;
    const int64_t waves = (int64_t)gridDim.x * 4;
    const int lane = threadIdx.x & 63;
    for (int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); w < N * segments; w += waves) {
        const int64_t n = w / segments;
        const int64_t j0 = (w - n * segments) * 256 + lane;
        const uint32_t row = sort_key(ids[n], range);
        const bool found = row < range.rows;
        vec v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t j = j0 + u * 64;
            if (found && j * V < D)
                v[u] = *reinterpret_cast<const vec*>(table + (int64_t)row * ld + vec_col<V>(j, D));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t j = j0 + u * 64;
            if (j * V >= D) break;
            float f[V];
            unpack<T, V>(v[u], f);
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = found ? f[k] * scale : 0.f;
            store_cols<T, V>(out + n * D + vec_col<V>(j, D), f);
        }
    }
}

// ---------------------------------------------------------------------------
// gradient: clear and sort
// ---------------------------------------------------------------------------
struct Fill { void* rows; int64_t bytes; uint8_t* touched; int64_t n_touched; };

// Lane `t` of `n` lanes clears its share.
__device__ __forceinline__ void clear(const Fill& F, int64_t t, int64_t n) {
    typedef uint32_t q __attribute__((ext_vector_type(4), aligned(2)));
    const int64_t quads = F.bytes >> 4;
    for (int64_t i = t; i < quads; i += n) reinterpret_cast<q*>(F.rows)[i] = q{0, 0, 0, 0};
    uint16_t* tail = reinterpret_cast<uint16_t*>(F.rows) + quads * 8;
    for (int64_t i = t; i < ((F.bytes & 15) >> 1); i += n) tail[i] = 0;
    for (int64_t i = t; i < F.n_touched; i += n) F.touched[i] = 0;
}

__global__ __launch_bounds__(256) void row_clear_kernel(Fill F) {
    clear(F, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// Workgroup 0 sorts up to ITEMS * 1024 ids; the others clear.  The ranking is that of the tile
// scatter (radix_sort.hpp), with sixteen waves and the pairs in registers between the passes.
template <typename I, int ITEMS>
__global__ __launch_bounds__(1024) void row_sort_small_kernel(const I* __restrict__ ids, int N,
                                                              IdRange range, int bits,
                                                              uint32_t* __restrict__ keys_out,
                                                              uint32_t* __restrict__ vals_out,
                                                              Fill F) {
    __shared__ uint32_t lkey[ITEMS * 1024];
    __shared__ uint16_t lval[ITEMS * 1024];
    __shared__ uint16_t wcount[16][kRadix];      // a wave holds at most 64 * ITEMS <= 1024 of a digit
    __shared__ uint32_t digit_base[kRadix];
    __shared__ uint32_t wsum[4];
    if (blockIdx.x > 0) {
        clear(F, (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x, (int64_t)(gridDim.x - 1) * 1024);
        return;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t lt_mask = lane == 0 ? 0ull : (~0ull >> (64 - lane));
    const int wbase = w * (ITEMS * 64);
    uint32_t key[ITEMS];
    uint16_t val[ITEMS], rank[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = wbase + r * 64 + lane;
        key[r] = i < N ? sort_key(ids[i], range) : ~0u;
        val[r] = (uint16_t)i;
    }
    for (int shift = 0; shift < bits; shift += kRadixBits) {
        const int nbits = min(kRadixBits, bits - shift);
        for (int k = threadIdx.x; k < 16 * kRadix; k += 1024) (&wcount[0][0])[k] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            // (positions behind N are the last ones of the array and hold the largest key: they
            // keep their place behind every id in every pass)
            const bool valid = wbase + r * 64 + lane < N;
            const uint32_t d = digit_of(key[r], shift);
            uint64_t peers = __ballot(valid);
#pragma unroll
            for (int b = 0; b < kRadixBits; ++b) {
                if (b < nbits) {
                    const uint64_t m = __ballot((d >> b) & 1u);
                    peers &= ((d >> b) & 1u) ? m : ~m;
                }
            }
            const uint32_t before = wcount[w][d];
            const uint32_t below = __popcll(peers & lt_mask);
            rank[r] = (uint16_t)(before + below);
            __builtin_amdgcn_wave_barrier();
            if (valid && below == 0) wcount[w][d] = (uint16_t)(before + __popcll(peers));
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        uint32_t run = 0;
        if (threadIdx.x < kRadix) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const uint32_t c = wcount[k][threadIdx.x];
                wcount[k][threadIdx.x] = (uint16_t)run;
                run += c;
            }
            const uint32_t inc = wave_scan_incl(run);
            if (lane == 63) wsum[w] = inc;
            digit_base[threadIdx.x] = inc - run;
        }
        __syncthreads();
        if (threadIdx.x < kRadix) {
            uint32_t off = 0;
            for (int k = 0; k < w; ++k) off += wsum[k];
            digit_base[threadIdx.x] += off;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            if (wbase + r * 64 + lane < N) {
                const uint32_t d = digit_of(key[r], shift);
                const uint32_t p = digit_base[d] + wcount[w][d] + rank[r];
                lkey[p] = key[r];
                lval[p] = val[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            const int i = wbase + r * 64 + lane;
            if (i < N) { key[r] = lkey[i]; val[r] = lval[i]; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = wbase + r * 64 + lane;
        if (i < N) { keys_out[i] = key[r]; vals_out[i] = val[r]; }
    }
}

// ---------------------------------------------------------------------------
// gradient: sums over runs of equal ids
// ---------------------------------------------------------------------------
struct Segments {
    const uint32_t* keys;     // sorted row numbers, `rows` and above = no row
    const uint32_t* pos;      // positions of their ids
    int N;
    uint32_t rows;
    int64_t D, ld;            // columns; elements between gradient rows
    int lg;                   // lanes per group = 2^lg
    int per_group;            // sorted positions per lane group
    float scale;
    uint8_t* touched;
    float* partial;           // [piece][2][D]: {run from an earlier piece, run into the next}
};

template <int V>
__device__ __forceinline__ void store_partial(float* __restrict__ p, const float f[V]) {
    if constexpr (V == 8) store_cols<float, 8>(p, f);
    else store_cols<float, V>(p, f);
}

template <typename T, typename O, int V>
__global__ __launch_bounds__(256) void row_segment_kernel(Segments S, const T* __restrict__ grad,
                                                          O* __restrict__ out) {
    typedef typename VecOf<T, V>::type vec;
    __shared__ uint32_t skey[kPieceMax + 2];          // with the key before and behind the piece
    __shared__ uint32_t spos[kPieceMax];
    __shared__ float sval[256 * V];                   // open sums, lane-contiguous per component
    __shared__ uint8_t sopen[256];                    // group's open sum reaches its left edge
    constexpr uint32_t kNone = ~0u;                   // no such key: rows < 2^31
    const int lanes = 1 << S.lg, n_groups = 256 >> S.lg;
    const int g = threadIdx.x >> S.lg;
    const int64_t j = (int64_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    const bool col_ok = j * V < S.D;
    const int64_t c = col_ok ? vec_col<V>(j, S.D) : 0;
    const int piece = n_groups * S.per_group;
    const int64_t base = (int64_t)blockIdx.x * piece;
    const int len = (int)min((int64_t)piece, (int64_t)S.N - base);
    for (int i = threadIdx.x; i < len + 2; i += 256) {
        const int64_t q = base + i - 1;
        skey[i] = q >= 0 && q < S.N ? S.keys[q] : kNone;
    }
    for (int i = threadIdx.x; i < len; i += 256) spos[i] = S.pos[base + i];
    __syncthreads();

    const int first = min(g * S.per_group, len), last = min(first + S.per_group, len);
    float acc[V], head[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = head[k] = 0.f;
    uint32_t cur = kNone;
    bool from_left = false;            // the run being summed began before this group's positions
    bool has_head = false, has_tail = false;
    uint32_t head_key = kNone;

    auto write_row = [&](uint32_t row, const float f[V]) {
        if (row >= S.rows || !col_ok) return;
        float o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = f[k] * S.scale;
        store_cols<O, V>(out + (int64_t)row * S.D + c, o);
    };
    auto close_run = [&] {
        if (from_left) {
            has_head = true; head_key = cur;
#pragma unroll
            for (int k = 0; k < V; ++k) head[k] = acc[k];
        } else {
            write_row(cur, acc);
        }
    };

    if (first < last) {
        cur = skey[first + 1];
        from_left = skey[first] == cur;
        auto begin_row = [&](uint32_t row) {
            if (S.touched && row < S.rows && j == 0) S.touched[row] = 1;
        };
        if (!from_left) begin_row(cur);
        constexpr int U = 4;
        for (int i0 = first; i0 < last; i0 += U) {
            vec v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u;
                if (i < last && col_ok && skey[i + 1] < S.rows)
                    v[u] = *reinterpret_cast<const vec*>(grad + (int64_t)spos[i] * S.ld + c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u;
                if (i >= last) break;
                const uint32_t k_i = skey[i + 1];
                if (k_i != cur) {
                    close_run();
                    cur = k_i; from_left = false;
                    begin_row(cur);
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] = 0.f;
                }
                if (col_ok && k_i < S.rows) {
                    float f[V];
                    unpack<T, V>(v[u], f);
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] += f[k];
                }
            }
        }
        if (skey[last + 1] == cur) has_tail = true; else close_run();
    }

    // Open sums: inclusive scan over the groups, where a group whose positions are one single
    // run that came from the left adds its left neighbour's.
    bool open = has_tail && from_left;
    const int l = threadIdx.x;
#pragma unroll
    for (int k = 0; k < V; ++k) sval[k * 256 + l] = acc[k];
    sopen[l] = open;
    __syncthreads();
    for (int s = 1; s < n_groups; s <<= 1) {
        const int q = l - (s << S.lg);
        const bool add = open && q >= 0;
        float t[V];
        bool o = open;
        if (add) {
            o = sopen[q];
#pragma unroll
            for (int k = 0; k < V; ++k) t[k] = sval[k * 256 + q];
        }
        __syncthreads();
        if (add) {
#pragma unroll
            for (int k = 0; k < V; ++k) sval[k * 256 + l] = acc[k] = t[k] + acc[k];
            sopen[l] = open = o;
        }
        __syncthreads();
    }
    // (open now: the run fills everything from the workgroup's left edge to this group's end)
    if (has_head) {
        bool before_piece = true;
        if (g > 0) {
            const int q = l - lanes;
            before_piece = sopen[q];
#pragma unroll
            for (int k = 0; k < V; ++k) head[k] += sval[k * 256 + q];
        }
        if (!before_piece) write_row(head_key, head);
        else if (col_ok && head_key < S.rows)
            store_partial<V>(S.partial + ((int64_t)blockIdx.x * 2) * S.D + c, head);
    }
    if (has_tail && last == len && cur < S.rows && col_ok)
        store_partial<V>(S.partial + ((int64_t)blockIdx.x * 2 + (open ? 0 : 1)) * S.D + c, acc);
}

// One workgroup per piece and column segment; those in whose piece no run begins that goes on
// into the next one end at once.
template <typename O, int V>
__global__ __launch_bounds__(256) void row_join_kernel(Segments S, O* __restrict__ out, int n_pieces) {
    __shared__ float sval[256 * V];
    const int lanes = 1 << S.lg, n_groups = 256 >> S.lg;
    const int64_t piece = (int64_t)n_groups * S.per_group;
    const int b = blockIdx.x;
    const int64_t base = b * piece, end = base + piece;       // (the last piece is not launched)
    const uint32_t k = S.keys[end];
    if (k >= S.rows || S.keys[end - 1] != k || (b > 0 && S.keys[base - 1] == k)) return;
    // pieces whose first id is k: b + 1 .. b + count
    int count = 0;
    for (;;) {
        const int64_t p = (int64_t)b + 1 + count + threadIdx.x;
        const int found = __syncthreads_count(p < n_pieces && S.keys[p * piece] == k);
        count += found;
        if (found < 256) break;
    }
    const int g = threadIdx.x >> S.lg;
    const int64_t j = (int64_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    const bool col_ok = j * V < S.D;
    const int64_t c = col_ok ? vec_col<V>(j, S.D) : 0;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    if (col_ok) {
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = S.partial[((int64_t)b * 2 + 1) * S.D + c + i];
        }
#pragma unroll 4
        for (int p = 1 + g; p <= count; p += n_groups) {
            const float* q = S.partial + ((int64_t)(b + p) * 2) * S.D + c;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += q[i];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sval[i * 256 + threadIdx.x] = acc[i];
    for (int s = n_groups >> 1; s > 0; s >>= 1) {
        __syncthreads();
        if (g < s) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                acc[i] += sval[i * 256 + threadIdx.x + (s << S.lg)];
                sval[i * 256 + threadIdx.x] = acc[i];
            }
        }
    }
    if (g == 0 && col_ok) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= S.scale;
        store_cols<O, V>(out + (int64_t)k * S.D + c, acc);
    }
}

namespace {

int ceil_log2(int64_t x) { int l = 0; while (((int64_t)1 << l) < x) ++l; return l; }

// How the gradient is cut up: by the number of ids, columns and the vector width alone.
struct SegmentPlan { int vec, lg, per_group, pieces, segments; };
SegmentPlan plan_segments(int64_t N, int64_t D, int type) {
    SegmentPlan p;
    const int full = type == ELEM_F32 ? 4 : 8;
    p.vec = D >= full ? full : 1;
    const int64_t vectors = (D + p.vec - 1) / p.vec;
    p.lg = vectors >= 64 ? 6 : ceil_log2(vectors);
    p.segments = (int)((vectors + (1 << p.lg) - 1) >> p.lg);
    const int groups = 256 >> p.lg;
    // about 2048 workgroups (eight per CU) where there are enough ids; 4 positions at least (the
    // loads a lane keeps in flight), 64 at most (what one float32 sum may run over)
    int64_t per = N * p.segments / ((int64_t)groups * 2048);
    p.per_group = 4;
    while (p.per_group < per && p.per_group < 64 && groups * p.per_group < kPieceMax) p.per_group *= 2;
    // (a piece of few groups still takes a few dozen ids: fewer partial rows to join)
    const int piece = groups * p.per_group;
    p.pieces = (int)((N + piece - 1) / piece);
    return p;
}

struct GradWorkspace {
    uint32_t *key[2], *val[2], *thist, *totals;
    float* partial;
    size_t bytes;
};
GradWorkspace carve_grad(void* ws, int64_t N, int64_t D, int type) {
    GradWorkspace w;
    char* p = (char*)ws;
    size_t off = 0;
    auto take = [&](size_t bytes) { char* q = p + off; off += align256(bytes); return q; };
    const bool tiles = N > kLdsSortMax;
    for (int i = 0; i < 2; ++i) {
        const bool need = i == 0 || tiles;
        w.key[i] = (uint32_t*)take(need ? 4 * (size_t)N : 0);
        w.val[i] = (uint32_t*)take(need ? 4 * (size_t)N : 0);
    }
    const size_t ntiles = ((size_t)N + kSortTile - 1) / kSortTile;
    w.thist = (uint32_t*)take(tiles ? 4 * kRadix * ntiles : 0);
    w.totals = (uint32_t*)take(tiles ? 4 * kRadix : 0);
    const SegmentPlan s = plan_segments(N, D, type);
    w.partial = (float*)take(s.pieces > 1 ? sizeof(float) * 2 * (size_t)s.pieces * D : 0);
    w.bytes = off;
    return w;
}

template <typename I>
int sort_small(const I* ids, int N, IdRange range, int bits, const GradWorkspace& w, const Fill& F,
               int clear_blocks, hipStream_t s) {
    const int grid = 1 + clear_blocks;
    if (N <= 1024) row_sort_small_kernel<I, 1><<<grid, 1024, 0, s>>>(ids, N, range, bits, w.key[0], w.val[0], F);
    else if (N <= 4096) row_sort_small_kernel<I, 4><<<grid, 1024, 0, s>>>(ids, N, range, bits, w.key[0], w.val[0], F);
    else row_sort_small_kernel<I, 16><<<grid, 1024, 0, s>>>(ids, N, range, bits, w.key[0], w.val[0], F);
    VINGS_LAUNCH_CHECK();
    return VINGS_OK;
}

// Leaves the sorted pairs in key[*at], val[*at].
template <typename I>
int sort_tiles(const I* ids, int64_t N, IdRange range, int bits, const GradWorkspace& w, int* at,
               hipStream_t s) {
    const int ntiles = cdiv(N, kSortTile);
    int cur = 1;
    for (int shift = 0; shift < bits; shift += kRadixBits) {
        const int nbits = std::min(kRadixBits, bits - shift);
        if (shift == 0)
            sort_tile_hist_kernel<I><<<ntiles, kSortThreads, 0, s>>>(ids, N, 0, ntiles, w.thist, nullptr, range);
        else
            sort_tile_hist_kernel<uint32_t><<<ntiles, kSortThreads, 0, s>>>(w.key[cur], N, shift, ntiles, w.thist,
                                                                            nullptr, range);
        VINGS_LAUNCH_CHECK();
        sort_scan_kernel<<<kRadix, 256, 0, s>>>(w.thist, ntiles, w.totals);
        VINGS_LAUNCH_CHECK();
        if (shift == 0)
            sort_scatter_kernel<I><<<ntiles, kSortThreads, 0, s>>>(ids, nullptr, w.key[cur ^ 1], w.val[cur ^ 1], N, 0,
                                                                   ntiles, w.thist, w.totals, nullptr, nbits, range);
        else
            sort_scatter_kernel<uint32_t><<<ntiles, kSortThreads, 0, s>>>(w.key[cur], w.val[cur], w.key[cur ^ 1],
                                                                          w.val[cur ^ 1], N, shift, ntiles, w.thist,
                                                                          w.totals, nullptr, nbits, range);
        VINGS_LAUNCH_CHECK();
        cur ^= 1;
    }
    *at = cur;
    return VINGS_OK;
}

template <typename T, typename O, int V>
int segment_launches(const Segments& S, const SegmentPlan& p, const void* grad, void* out, hipStream_t s) {
    row_segment_kernel<T, O, V><<<dim3(p.pieces, p.segments), 256, 0, s>>>(S, (const T*)grad, (O*)out);
    VINGS_LAUNCH_CHECK();
    if (p.pieces > 1) {
        row_join_kernel<O, V><<<dim3(p.pieces - 1, p.segments), 256, 0, s>>>(S, (O*)out, p.pieces);
        VINGS_LAUNCH_CHECK();
    }
    return VINGS_OK;
}

template <typename T, typename O>
int segment_by_width(const Segments& S, const SegmentPlan& p, const void* grad, void* out, hipStream_t s) {
    return p.vec == 1 ? segment_launches<T, O, 1>(S, p, grad, out, s)
                      : segment_launches<T, O, Elem<T>::kVec>(S, p, grad, out, s);
}

template <typename T, typename I>
int lookup_impl(int64_t N, int64_t D, const void* table, int64_t ld, const void* ids, IdRange range,
                float scale, void* out, hipStream_t s) {
    constexpr int V = Elem<T>::kVec;
    const int64_t vectors = D >= V ? (D + V - 1) / V : D;
    if (vectors > 64) {
        const int segments = (int)((vectors + 255) / 256);
        const int64_t blocks = (N * segments + 3) / 4;
        row_lookup_wide_kernel<T, I><<<(int)std::min<int64_t>(blocks, 16384), 256, 0, s>>>(
            N, D, segments, (const T*)table, ld, (const I*)ids, range, scale, (T*)out);
    } else {
        const int lg = ceil_log2(vectors);
        const int64_t blocks = (N + 4 * (256 >> lg) - 1) / (4 * (256 >> lg));
        const int grid = (int)std::min<int64_t>(blocks, 16384);
        if (D >= V)
            row_lookup_kernel<T, I, V><<<grid, 256, 0, s>>>(N, D, (const T*)table, ld, (const I*)ids, range, scale, (T*)out, lg);
        else
            row_lookup_kernel<T, I, 1><<<grid, 256, 0, s>>>(N, D, (const T*)table, ld, (const I*)ids, range, scale, (T*)out, lg);
    }
    VINGS_LAUNCH_CHECK();
    return VINGS_OK;
}

template <typename T>
int lookup_by_id(int id_bytes, int64_t N, int64_t D, const void* table, int64_t ld, const void* ids,
                 IdRange range, float scale, void* out, hipStream_t s) {
    return id_bytes == 8 ? lookup_impl<T, int64_t>(N, D, table, ld, ids, range, scale, out, s)
                         : lookup_impl<T, int32_t>(N, D, table, ld, ids, range, scale, out, s);
}

int check_shape(int64_t N, int64_t V, int64_t D, int type, int id_bytes) {
    VINGS_REQUIRE(N >= 0 && V >= 0 && D > 0, "sizes");
    VINGS_REQUIRE(N < ((int64_t)1 << 31) && V < ((int64_t)1 << 31) - 1 && D < ((int64_t)1 << 22),
                  "ids and rows must fit 31 bits, columns 22");
    VINGS_REQUIRE(elem_known(type), "element type");
    VINGS_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids are int32 or int64");
    return VINGS_OK;
}

}  // namespace
}  // namespace vings

using namespace vings;

extern "C" int vings_row_lookup(int64_t n_ids, int64_t n_rows, int64_t n_cols, const void* table,
                                int64_t table_stride, int type, const void* ids, int id_bytes,
                                float scale, void* out, void* stream) {
    const int rc = check_shape(n_ids, n_rows, n_cols, type, id_bytes);
    if (rc != VINGS_OK) return rc;
    if (n_ids == 0) return VINGS_OK;
    VINGS_REQUIRE((table || n_rows == 0) && ids && out, "null pointer");
    VINGS_REQUIRE(table_stride >= n_cols || n_rows <= 1, "rows must not overlap");
    VINGS_REQUIRE((((uintptr_t)table | (uintptr_t)out) & (elem_bytes(type) - 1)) == 0 &&
                      ((uintptr_t)ids & (id_bytes - 1)) == 0, "element alignment");
    hipStream_t s = (hipStream_t)stream;
    // (every row may be looked up, a padding row too: only its gradient is withheld)
    const IdRange range{(uint32_t)n_rows, -1};
    ProfScope prof(PROF_AUX, s);
    if (type == ELEM_F32)
        return lookup_by_id<float>(id_bytes, n_ids, n_cols, table, table_stride, ids, range, scale, out, s);
    if (type == ELEM_BF16)
        return lookup_by_id<__bf16>(id_bytes, n_ids, n_cols, table, table_stride, ids, range, scale, out, s);
    return lookup_by_id<_Float16>(id_bytes, n_ids, n_cols, table, table_stride, ids, range, scale, out, s);
}

extern "C" size_t vings_row_lookup_backward_workspace_bytes(int64_t n_ids, int64_t n_cols, int type) {
    if (n_ids <= 0 || n_cols <= 0 || n_ids >= ((int64_t)1 << 31) || !elem_known(type)) return 0;
    return carve_grad(nullptr, n_ids, n_cols, type).bytes;
}

extern "C" int vings_row_lookup_backward(int64_t n_ids, int64_t n_rows, int64_t n_cols,
                                         const void* grad, int64_t grad_stride, int type,
                                         const void* ids, int id_bytes, int64_t padding_id,
                                         float scale, void* rows, int rows_type, uint8_t* touched,
                                         int keep_touched, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    const int rc = check_shape(n_ids, n_rows, n_cols, type, id_bytes);
    if (rc != VINGS_OK) return rc;
    VINGS_REQUIRE(rows_type == type || rows_type == ELEM_F32, "rows have the gradient's type or float32");
    if (n_rows == 0) return VINGS_OK;
    VINGS_REQUIRE(rows, "null pointer");
    VINGS_REQUIRE(((uintptr_t)rows & (elem_bytes(rows_type) - 1)) == 0, "element alignment");
    hipStream_t s = (hipStream_t)stream;
    const Fill F{rows, n_rows * n_cols * elem_bytes(rows_type), touched, touched && !keep_touched ? n_rows : 0};
    // clearing: 64 KB per workgroup, eight workgroups per CU at most
    const int64_t per = 65536;
    int clear_blocks = (int)std::min<int64_t>(2048, (F.bytes + F.n_touched + per - 1) / per);
    ProfScope prof(PROF_AUX, s);
    if (n_ids == 0) {
        row_clear_kernel<<<clear_blocks, 256, 0, s>>>(F);
        VINGS_LAUNCH_CHECK();
        return VINGS_OK;
    }
    VINGS_REQUIRE(grad && ids && workspace, "null pointer");
    VINGS_REQUIRE(grad_stride >= 0, "sizes");
    VINGS_REQUIRE(((uintptr_t)grad & (elem_bytes(type) - 1)) == 0 && ((uintptr_t)ids & (id_bytes - 1)) == 0,
                  "element alignment");
    VINGS_REQUIRE(((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
    const GradWorkspace w = carve_grad(workspace, n_ids, n_cols, type);
    if (workspace_bytes < w.bytes) {
        set_error("row gradient workspace too small: %zu < %zu", workspace_bytes, w.bytes);
        return VINGS_ERR_CAPACITY;
    }
    const IdRange range{(uint32_t)n_rows, padding_id};
    const int bits = std::max(1, bits_for((uint32_t)n_rows));
    int at = 0, rs;
    if (n_ids <= kLdsSortMax) {
        rs = id_bytes == 8 ? sort_small((const int64_t*)ids, (int)n_ids, range, bits, w, F, clear_blocks, s)
                           : sort_small((const int32_t*)ids, (int)n_ids, range, bits, w, F, clear_blocks, s);
    } else {
        row_clear_kernel<<<clear_blocks, 256, 0, s>>>(F);
        VINGS_LAUNCH_CHECK();
        rs = id_bytes == 8 ? sort_tiles((const int64_t*)ids, n_ids, range, bits, w, &at, s)
                           : sort_tiles((const int32_t*)ids, n_ids, range, bits, w, &at, s);
    }
    if (rs != VINGS_OK) return rs;
    const SegmentPlan p = plan_segments(n_ids, n_cols, type);
    const Segments S{w.key[at], w.val[at], (int)n_ids, (uint32_t)n_rows, n_cols, grad_stride, p.lg,
                     p.per_group, scale, touched, w.partial};
    if (type == ELEM_F32) return segment_by_width<float, float>(S, p, grad, rows, s);
    if (type == ELEM_BF16)
        return rows_type == ELEM_F32 ? segment_by_width<__bf16, float>(S, p, grad, rows, s)
                                     : segment_by_width<__bf16, __bf16>(S, p, grad, rows, s);
    return rows_type == ELEM_F32 ? segment_by_width<_Float16, float>(S, p, grad, rows, s)
                                 : segment_by_width<_Float16, _Float16>(S, p, grad, rows, s);
}
