// Rows of a table by integer id, scaled, and the gradient of that table, on gfx950.
//
//   lookup     out[n] = scale * table[id[n]]                     (zeros where id[n] names no row)
//   gradient   dtable[v] = scale * sum over {n : id[n] = v} of g[n],   touched[v] = any such n
//
// Both are HBM-bound.  The lookup is one gather: a wave takes a row (or several short ones, a
// lane group each) with 16-byte accesses, four in flight per lane: 16381 rows of 2048 bfloat16 in
// 21 us, a million rows of 12 float32 in 12 us, both 4.9 TB/s of what has to move.
//
// The gradient sums by SORTED ids, with no float atomics, so its bits do not depend on timing:
//   1. the ids and their positions are ordered by a stable radix sort; ids that name no row sort
//      behind the last row.  Up to 32768 ids workgroups sort runs of 1024 in LDS and a second
//      launch merges the runs, every id finding its place by bisection in each of them, while
//      further workgroups of both launches clear dtable and touched; more ids take the tile
//      passes of radix_sort.hpp, 8 bits each (clearing beside the first; 100 k ids into 60 k rows
//      of 16 float32: 42 us with clearing and every scan in launches of their own, now 36)
//   2. segment kernel: the sorted positions are cut into pieces of equal length, whatever rows
//      they belong to, so one frequent id costs no more than many rare ones.  A lane group walks
//      a few consecutive positions, holds its columns' sum in float32 registers, and writes a
//      row whenever a run of equal ids begins and ends inside its piece
//   3. runs that cross lane groups are joined in LDS by a segmented scan over the groups (in
//      sorted order the run of group g continues that of group g - s exactly if their last and
//      first ids are equal), runs that cross workgroups leave one partial row per workgroup
//   4. join kernel: the workgroup in whose piece such a run begins adds the partial rows of the
//      pieces behind it, in a fixed tree
// Few rows of few columns under many ids (per-keyframe rows) need no global order at all: a
// workgroup sorts 1024 ids in LDS, sums their runs as in 2 and 3 and leaves one partial row per
// row it met; a second launch adds those over the workgroups.  The gradient is then read in
// stretches of 1024 rows instead of all over, and two launches replace seven (one, up to 1024 ids).
// Sums are float32: at most 64 terms in a row in a lane group, then the scan, then the partial rows
// of a run dealt out over the lane groups of its join; the result is scaled and rounded once.
// Measured: 16381 ids into 32768 rows of 2048 bfloat16 in 58 us, of which the two sorting launches
// 24 (they clear 134 MB meanwhile, at 5.6 TB/s), segments 24, join 6; a million ids into 80 rows of
// 12 float32 in 23 us (local sums 19: 2 us of latency for each of ids, ranking and rows, then 56 MB
// at 4.7 TB/s; join 4).
//
// Serves per-keyframe rows that every splat reads through the keyframe that owns it
// (globalkf_id, /root/reference/scripts/gaussian/gaussian_model.py:163-168) and any wide table;
// the reference itself has no learned table.
#include <algorithm>

#include "elem_types.hpp"
#include "radix_sort.hpp"

namespace vings {

constexpr int kRun = 1024;                // ids a workgroup sorts in LDS
constexpr int kMaxRuns = 32;              // runs the merge launch takes
constexpr int kMergeSortMax = kRun * kMaxRuns;
constexpr int kTileThreads = 512;         // few-rows form: lanes and
constexpr int kTileIds = 1024;            // ids per workgroup
constexpr int kTileItems = kTileIds / kTileThreads;
constexpr int kFewRows = 4095;            // ... 12-bit keys, the one of ids without a row included
constexpr int kFewTiles = 4096;           // ... partial rows that its join adds, at most
constexpr int kPieceMax = 2048;           // sorted positions per workgroup of the segment kernel
constexpr int64_t kMaxStride = 1 << 20;   // elements between gradient rows: byte offsets inside a
static_assert(kMaxStride * 4 * (kTileIds - 1) < ((int64_t)1 << 32), "32-bit offsets");   // tile fit

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

// A row per lane group of 2^lg lanes, four rows at a time; rows of up to 64 vectors.
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

// The first pass's histograms in workgroups [0, ntiles), the others clear.
template <typename I, bool DIRECT>
__global__ __launch_bounds__(kSortThreads) void row_first_hist_kernel(const I* __restrict__ ids, int64_t N, int ntiles,
                                                                      uint32_t* __restrict__ thist, IdRange range,
                                                                      Fill F) {
    if ((int)blockIdx.x >= ntiles)
        clear(F, (int64_t)(blockIdx.x - ntiles) * kSortThreads + threadIdx.x,
              (int64_t)(gridDim.x - ntiles) * kSortThreads);
    else
        sort_tile_hist<I, DIRECT>(ids, N, 0, ntiles, thist, range);
}

// Stable counting sort of one digit inside a workgroup: the place of this lane's ITEMS keys
// (item r of lane l of wave w is key number (w * ITEMS + r) * 64 + l) among the workgroup's
// `count` valid keys.  Ranking as in the tile scatter (radix_sort.hpp).  counts: [WAVES][256],
// base: [256], both LDS; on return base[d] is the number of keys with a smaller digit.
template <int WAVES, int ITEMS>
__device__ __forceinline__ void block_digit_places(const uint32_t key[ITEMS], int count, int shift, int nbits,
                                                   uint16_t (*counts)[kRadix], uint32_t* base,
                                                   uint32_t* wsum, uint32_t place[ITEMS]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t lt_mask = lane == 0 ? 0ull : (~0ull >> (64 - lane));
    for (int k = threadIdx.x; k < WAVES * kRadix; k += WAVES * 64) (&counts[0][0])[k] = 0;
    __syncthreads();
    // which lanes hold the same digit: independent for the items, then one chain of counters
    uint32_t below[ITEMS], peers_n[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const bool valid = (w * ITEMS + r) * 64 + lane < count;
        const uint32_t d = digit_of(key[r], shift);
        uint64_t peers = __ballot(valid);
#pragma unroll
        for (int b = 0; b < kRadixBits; ++b) {
            if (b < nbits) {
                const uint64_t m = __ballot((d >> b) & 1u);
                peers &= ((d >> b) & 1u) ? m : ~m;
            }
        }
        below[r] = __popcll(peers & lt_mask);
        peers_n[r] = valid ? __popcll(peers) : 0u;
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint32_t d = digit_of(key[r], shift);
        const uint32_t before = counts[w][d];
        place[r] = before + below[r];
        __builtin_amdgcn_wave_barrier();
        if (peers_n[r] && below[r] == 0) counts[w][d] = (uint16_t)(before + peers_n[r]);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    uint32_t run = 0, inc = 0;
    const int d = threadIdx.x;
    if (d < kRadix) {
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const uint32_t c = counts[k][d];
            counts[k][d] = (uint16_t)run;
            run += c;
        }
        inc = wave_scan_incl(run);
        if (lane == 63) wsum[w] = inc;
    }
    __syncthreads();
    if (d < kRadix) {
        uint32_t off = inc - run;
        for (int k = 0; k < w; ++k) off += wsum[k];
        base[d] = off;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint32_t k = digit_of(key[r], shift);
        place[r] += base[k] + counts[w][k];
    }
}

// Workgroups [0, n_runs) sort 1024 ids each, the others clear.
template <typename I>
__global__ __launch_bounds__(1024) void row_sort_runs_kernel(const I* __restrict__ ids, int N, int n_runs,
                                                             IdRange range, int bits,
                                                             uint32_t* __restrict__ keys_out,
                                                             uint32_t* __restrict__ vals_out, Fill F) {
    __shared__ uint16_t counts[16][kRadix];
    __shared__ uint32_t base[kRadix], wsum[4];
    __shared__ uint32_t lkey[kRun];
    __shared__ uint32_t lval[kRun];
    if ((int)blockIdx.x >= n_runs) {
        clear(F, (int64_t)(blockIdx.x - n_runs) * 1024 + threadIdx.x, (int64_t)(gridDim.x - n_runs) * 1024);
        return;
    }
    const int first = blockIdx.x * kRun, t = threadIdx.x;
    const int count = min(kRun, N - first);
    uint32_t key[1] = {t < count ? sort_key(ids[first + t], range) : ~0u};
    uint32_t val = (uint32_t)(first + t);
    for (int shift = 0; shift < bits; shift += kRadixBits) {
        uint32_t place[1];
        block_digit_places<16, 1>(key, count, shift, min(kRadixBits, bits - shift), counts, base, wsum, place);
        if (t < count) { lkey[place[0]] = key[0]; lval[place[0]] = val; }
        __syncthreads();
        if (t < count) { key[0] = lkey[t]; val = lval[t]; }
        __syncthreads();
    }
    if (t < count) { keys_out[first + t] = key[0]; vals_out[first + t] = val; }
}

// Merges up to kMaxRuns sorted runs: the place of an id is its place in its own run plus, for
// every earlier run, the ids there that are not larger, and for every later one those that are
// smaller.  All keys sit in LDS; four bisections of a lane run side by side.
// (RUNS: the LDS that the launch reserves, for its clearing workgroups too.)
constexpr int kMergeThreads = 256;
template <int RUNS>
__global__ __launch_bounds__(kMergeThreads) void row_merge_runs_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int N, int n_runs, int n_merge,
    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out, Fill F) {
    __shared__ __align__(16) uint32_t lkey[RUNS * kRun];
    if ((int)blockIdx.x >= n_merge) {
        clear(F, (int64_t)(blockIdx.x - n_merge) * kMergeThreads + threadIdx.x,
              (int64_t)(gridDim.x - n_merge) * kMergeThreads);
        return;
    }
    // (all loads in flight together: the launch is a chain of latencies)
    uint4 q[RUNS];
    static_assert(kRun == 4 * kMergeThreads, "a run is one round of 16-byte loads");
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
        // (a load that begins before N ends inside the array's 256-byte granule)
        const int i = r * kRun + 4 * threadIdx.x;
        q[r] = *reinterpret_cast<const uint4*>(keys + (i < N ? i : 0));
    }
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
        const int i = r * kRun + 4 * threadIdx.x;
        const uint4 k = make_uint4(i < N ? q[r].x : ~0u, i + 1 < N ? q[r].y : ~0u, i + 2 < N ? q[r].z : ~0u,
                                   i + 3 < N ? q[r].w : ~0u);
        if (r < n_runs) *reinterpret_cast<uint4*>(lkey + i) = k;
    }
    __syncthreads();
    const int e = blockIdx.x * kMergeThreads + threadIdx.x;
    if (e >= N) return;
    const uint32_t key = lkey[e];
    const int own = e / kRun;
    uint32_t place = (uint32_t)(e - own * kRun);
    for (int r0 = 0; r0 < n_runs; r0 += 4) {
        uint32_t pos[4] = {0, 0, 0, 0}, limit[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) limit[u] = key + (r0 + u < own ? 1u : 0u);
#pragma unroll
        for (int step = kRun / 2; step > 0; step >>= 1)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = min(r0 + u, n_runs - 1);
                if (lkey[r * kRun + pos[u] + step - 1] < limit[u]) pos[u] += step;
            }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = r0 + u;
            if (r < n_runs && r != own) place += pos[u] + (lkey[r * kRun + pos[u]] < limit[u] ? 1u : 0u);
        }
    }
    keys_out[place] = key;
    vals_out[place] = vals[e];
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
                              // few rows: [row][tile][D] with by_row, else [tile][run][D]
    bool by_row;
};

// Partial rows that a tile of the few-rows form leaves with numbered runs, at most.
__host__ __device__ __forceinline__ int64_t tile_runs(int64_t rows) { return rows < kTileIds ? rows : kTileIds; }

// Sums of the runs of equal keys among a workgroup's `len` sorted positions.  skey[1 .. len]: the
// keys, skey[0] and skey[len + 1] those before and behind them (kNoKey where there are none);
// load(i): this lane's columns of the gradient row at position i.  Calls write(row, sum) for runs
// that lie inside, write_head(sum) for the one that began before, write_tail(sum, all) for the one
// that goes on behind (all: and began before), from the lanes that hold the sum's columns.
// A wave walks several groups at once and one of them closes a run at nearly every step, so a
// step has little to do beside its addition: the loads need no guard and the address of a row is
// one multiply-add.
constexpr uint32_t kNoKey = ~0u;                     // rows < 2^31
template <int V, int THREADS> struct RunShared {
    float val[THREADS * V];                          // open sums, lane-contiguous per component
    uint8_t open[THREADS];                           // a group's open sum reaches the left edge
};

template <typename T, int V, int THREADS, typename F, typename W, typename H, typename L>
__device__ __forceinline__ void sum_runs(const Segments& S, uint32_t limit, const uint32_t* skey, int len, bool col_ok,
                                         RunShared<V, THREADS>& sh, F load, W write, H write_head, L write_tail) {
    typedef typename VecOf<T, V>::type vec;
    const int lanes = 1 << S.lg, n_groups = THREADS >> S.lg;
    const int g = threadIdx.x >> S.lg;
    const int first = min(g * S.per_group, len), last = min(first + S.per_group, len);
    float acc[V], head[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = head[k] = 0.f;
    uint32_t cur = kNoKey, head_key = kNoKey;
    bool from_left = false;            // the run being summed began before this group's positions
    bool has_head = false, has_tail = false;
    auto close_run = [&] {
        if (from_left) {
            has_head = true; head_key = cur;
#pragma unroll
            for (int k = 0; k < V; ++k) head[k] = acc[k];
        } else if (col_ok) {
            write(cur, acc);
        }
    };
    // ids without a row (keys from `limit` on) are the last of the order: the walk ends before them
    int stop = last;
    while (stop > first && skey[stop] >= limit) --stop;
    constexpr int U = 4;
    auto batch = [&](int i0, int n) {              // n <= U positions from i0
        vec v[U];
        uint32_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + min(u, n - 1);      // (a short batch loads its last row again)
            v[u] = load(i);
            key[u] = skey[i + 1];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= n) break;
            if (key[u] != cur) {
                close_run();
                cur = key[u]; from_left = false;
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] = 0.f;
            }
            float f[V];
            unpack<T, V>(v[u], f);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += f[k];
        }
    };
    if (first < stop) {
        cur = skey[first + 1];
        from_left = skey[first] == cur;
        int i0 = first;
        for (; i0 + U <= stop; i0 += U) batch(i0, U);
        if (i0 < stop) batch(i0, stop - i0);
        if (skey[stop + 1] == cur) has_tail = true; else close_run();
    }

    // Open sums: inclusive scan over the groups, where a group whose positions are one single
    // run that came from the left adds its left neighbour's.
    bool open = has_tail && from_left;
    const int l = threadIdx.x;
#pragma unroll
    for (int k = 0; k < V; ++k) sh.val[k * THREADS + l] = acc[k];
    sh.open[l] = open;
    // (the vote at the loop's head goes through an LDS store of its own and a barrier behind that:
    // the wait for it there covers the stores of the round before)
    for (int s = 1; s < n_groups; s <<= 1) {
        const int q = l - (s << S.lg);
        const bool add = open && q >= 0;
        if (!__syncthreads_or(add)) break;
        float t[V];
        bool o = open;
        if (add) {
            o = sh.open[q];
#pragma unroll
            for (int k = 0; k < V; ++k) t[k] = sh.val[k * THREADS + q];
        }
        __syncthreads();
        if (add) {
#pragma unroll
            for (int k = 0; k < V; ++k) sh.val[k * THREADS + l] = acc[k] = t[k] + acc[k];
            sh.open[l] = open = o;
        }
    }
    __syncthreads();
    // (open now: the run fills everything from the workgroup's left edge to this group's end)
    if (has_head) {
        bool before_piece = true;
        if (g > 0) {
            const int q = l - lanes;
            before_piece = sh.open[q];
#pragma unroll
            for (int k = 0; k < V; ++k) head[k] += sh.val[k * THREADS + q];
        }
        if (col_ok) {
            if (before_piece) write_head(head); else write(head_key, head);
        }
    }
    if (has_tail && last == len && col_ok) write_tail(acc, open);
}

// Byte offset of row `row` of rows that lie `pitch` bytes apart.
__device__ __forceinline__ int64_t row_offset(uint32_t row, uint32_t pitch) { return (int64_t)((uint64_t)row * pitch); }

template <typename O, int V>
__device__ __forceinline__ void write_scaled(O* __restrict__ p, const float f[V], float scale) {
    float o[V];
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = f[k] * scale;
    store_cols<O, V>(p, o);
}

template <typename T, typename O, int V>
__global__ __launch_bounds__(256) void row_segment_kernel(Segments S, const T* __restrict__ grad,
                                                          O* __restrict__ out) {
    typedef typename VecOf<T, V>::type vec;
    extern __shared__ uint32_t smem[];                // (the usual piece takes a few hundred bytes)
    __shared__ RunShared<V, 256> sh;
    const int lanes = 1 << S.lg;
    const int64_t j = (int64_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    const bool col_ok = j * V < S.D;
    const int64_t c = col_ok ? vec_col<V>(j, S.D) : 0;
    const int piece = (256 >> S.lg) * S.per_group;
    uint32_t* skey = smem;                            // with the keys before and behind the piece
    uint32_t* spos = smem + piece + 2;
    const int64_t base = (int64_t)blockIdx.x * piece;
    const int len = (int)min((int64_t)piece, (int64_t)S.N - base);
    for (int i = threadIdx.x; i < len + 2; i += 256) {
        const int64_t q = base + i - 1;
        skey[i] = q >= 0 && q < S.N ? S.keys[q] : kNoKey;
    }
    for (int i = threadIdx.x; i < len; i += 256) spos[i] = S.pos[base + i];
    __syncthreads();
    float* partial = S.partial + (int64_t)blockIdx.x * 2 * S.D + c;
    const char* from = reinterpret_cast<const char*>(grad + c);
    char* to = reinterpret_cast<char*>(out + c);
    const uint32_t pitch = (uint32_t)S.ld * sizeof(T), out_pitch = (uint32_t)S.D * sizeof(O);
    uint8_t* touched = j == 0 ? S.touched : nullptr;
    sum_runs<T, V, 256>(
        S, S.rows, skey, len, col_ok, sh,
        [&](int i) { return *reinterpret_cast<const vec*>(from + row_offset(spos[i], pitch)); },
        [&](uint32_t row, const float* f) {
            write_scaled<O, V>(reinterpret_cast<O*>(to + row_offset(row, out_pitch)), f, S.scale);
            if (touched) touched[row] = 1;
        },
        [&](const float* f) { store_cols<float, V>(partial, f); },
        [&](const float* f, bool all) { store_cols<float, V>(partial + (all ? 0 : S.D), f); });
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
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = S.partial[((int64_t)b * 2 + 1) * S.D + c + i];
    }
    constexpr int U = 4;
    for (int p0 = 1 + g; p0 <= count; p0 += U * n_groups) {
        float f[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* q = S.partial + ((int64_t)(b + min(p0 + u * n_groups, count)) * 2) * S.D + c;
#pragma unroll
            for (int i = 0; i < V; ++i) f[u][i] = q[i];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += p0 + u * n_groups <= count ? f[u][i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sval[i * 256 + threadIdx.x] = acc[i];
    __syncthreads();
    for (int s = n_groups >> 1; s > 0; s >>= 1) {
        if (g < s) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                acc[i] += sval[i * 256 + threadIdx.x + (s << S.lg)];
                sval[i * 256 + threadIdx.x] = acc[i];
            }
        }
        __syncthreads();                              // (behind the stores, see row_tile_kernel)
    }
    if (g == 0 && col_ok) {
        write_scaled<O, V>(out + (int64_t)k * S.D + c, acc, S.scale);
        if (S.touched && j == 0) S.touched[k] = 1;
    }
}

// ---------------------------------------------------------------------------
// gradient, few rows: at most 4095 rows of at most 16 vectors
// ---------------------------------------------------------------------------
// The workgroup's own stable order of its 1024 ids, then their runs.  With one workgroup (ALONE) the
// sums are the rows themselves; otherwise they are partial rows.  Up to 256 rows those lie as the
// join reads them, partial[row][tile], and met[row][tile] says which there are; more rows would make
// that an array of holes and scattered stores, so the tile numbers its runs, run k goes to
// partial[tile][k] and met[tile][row] is k + 1, or 0 where the tile has no such id.
template <typename T, typename O, typename I, int V, bool ALONE>
__global__ __launch_bounds__(kTileThreads) void row_tile_kernel(Segments S, const T* __restrict__ grad,
                                                                const I* __restrict__ ids, IdRange range,
                                                                int bits, O* __restrict__ out,
                                                                uint16_t* __restrict__ met, int keep_touched) {
    typedef typename VecOf<T, V>::type vec;
    constexpr int kWaves = kTileThreads / 64;
    __shared__ uint16_t counts[kWaves][kRadix];
    __shared__ uint32_t base[kRadix], wsum[kWaves];
    __shared__ uint32_t skey[kTileIds + 2];           // keys, then the runs' numbers
    __shared__ uint32_t spos[kTileIds];               // positions, then byte offsets inside the tile
    __shared__ uint16_t smet[kFewRows + 1];
    __shared__ RunShared<V, kTileThreads> sh;
    const uint32_t pitch = (uint32_t)S.ld * sizeof(T);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * kTileIds;
    const int len = (int)min((int64_t)kTileIds, (int64_t)S.N - first);
    uint32_t key[kTileItems], pos[kTileItems], place[kTileItems];
#pragma unroll
    for (int r = 0; r < kTileItems; ++r) {
        pos[r] = (w * kTileItems + r) * 64 + lane;
        key[r] = sort_key(ids[first + min((int)pos[r], len - 1)], range);
    }
    for (uint32_t r = threadIdx.x; r < S.rows; r += kTileThreads) smet[r] = 0;
    if (threadIdx.x == 0) skey[0] = skey[len + 1] = kNoKey;
    for (int shift = 0; shift < bits; shift += kRadixBits) {
        if (shift) {                                  // the next digit, from the order so far
#pragma unroll
            for (int r = 0; r < kTileItems; ++r) {
                const int i = min((w * kTileItems + r) * 64 + lane, len - 1);
                key[r] = skey[i + 1];
                pos[r] = spos[i];
            }
            __syncthreads();
        }
        block_digit_places<kWaves, kTileItems>(key, len, shift, min(kRadixBits, bits - shift), counts, base, wsum,
                                               place);
#pragma unroll
        for (int r = 0; r < kTileItems; ++r)
            if ((w * kTileItems + r) * 64 + lane < len) { skey[place[r] + 1] = key[r]; spos[place[r]] = pos[r]; }
        // (here and not at the head of the next round: hipcc 7.2 leaves out the wait for LDS stores
        // in front of a barrier that is reached over a loop's back edge)
        __syncthreads();
    }
    uint32_t n_runs = S.rows;                         // (by_row: the keys stay the rows)
    if (ALONE || S.by_row) {
        for (int i = threadIdx.x; i < len; i += kTileThreads) {
            const uint32_t k = skey[i + 1];
            if (k < S.rows) smet[k] = 1;
            spos[i] *= pitch;
        }
    } else {
        // numbers of the runs: consecutive positions per lane, prefix sum of the runs beginning there
        uint32_t k[kTileItems], n_begin = 0;
        bool begins[kTileItems];
#pragma unroll
        for (int r = 0; r < kTileItems; ++r) {
            const int i = threadIdx.x * kTileItems + r;
            k[r] = i < len ? skey[i + 1] : kNoKey;
            begins[r] = k[r] < S.rows && k[r] != skey[min(i, len)];
            n_begin += begins[r];
        }
        const uint32_t inc = wave_scan_incl(n_begin);
        if (lane == 63) wsum[w] = inc;
        __syncthreads();
        uint32_t run = inc - n_begin;
        n_runs = 0;
#pragma unroll
        for (int q = 0; q < kWaves; ++q) {
            if (q < w) run += wsum[q];
            n_runs += wsum[q];
        }
#pragma unroll
        for (int r = 0; r < kTileItems; ++r) {
            const int i = threadIdx.x * kTileItems + r;
            run += begins[r];
            if (begins[r]) smet[k[r]] = (uint16_t)run;
            if (i < len) {
                skey[i + 1] = k[r] < S.rows ? run - 1 : kNoKey;
                spos[i] *= pitch;
            }
        }
    }
    __syncthreads();
    const int lanes = 1 << S.lg;
    const int64_t j = threadIdx.x & (lanes - 1);
    const bool col_ok = j * V < S.D;
    const int64_t c = col_ok ? vec_col<V>(j, S.D) : 0;
    const int64_t tiles = gridDim.x, tile = blockIdx.x;
    if (!ALONE) {
        const int64_t row_step = S.by_row ? tiles : 1, at = S.by_row ? tile : tile * S.rows;
        for (uint32_t r = threadIdx.x; r < S.rows; r += kTileThreads) met[at + r * row_step] = smet[r];
    } else {
        const float zero[V] = {};
        for (uint32_t r = threadIdx.x >> S.lg; r < S.rows; r += kTileThreads >> S.lg)
            if (col_ok && !smet[r]) store_cols<O, V>(out + (int64_t)r * S.D + c, zero);
        if (S.touched)
            for (uint32_t r = threadIdx.x; r < S.rows; r += kTileThreads)
                if (smet[r] || !keep_touched) S.touched[r] = smet[r] != 0;
    }
    const char* from = reinterpret_cast<const char*>(grad + first * S.ld + c);
    // where a sum goes: a row of the result, or a partial row (see Segments)
    char* to = ALONE ? reinterpret_cast<char*>(out + c)
                     : reinterpret_cast<char*>(S.partial + (S.by_row ? tile : tile * tile_runs(S.rows)) * S.D + c);
    const uint32_t step = (uint32_t)S.D * (ALONE ? (uint32_t)sizeof(O) : S.by_row ? 4u * (uint32_t)tiles : 4u);
    sum_runs<T, V, kTileThreads>(
        S, n_runs, skey, len, col_ok, sh, [&](int i) { return *reinterpret_cast<const vec*>(from + spos[i]); },
        [&](uint32_t k, const float* f) {
            char* q = to + row_offset(k, step);
            if constexpr (ALONE) write_scaled<O, V>(reinterpret_cast<O*>(q), f, S.scale);
            else store_cols<float, V>(reinterpret_cast<float*>(q), f);
        },
        [](const float*) {}, [](const float*, bool) {});
}

// One workgroup per row: its partial rows over the tiles, in a fixed tree.  The launch is two
// dependent loads per round whatever the rounds hold: many lanes for a row where there are few.
template <typename O, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void row_tile_join_kernel(Segments S, const uint16_t* __restrict__ met,
                                                                int tiles, O* __restrict__ out, int keep_touched) {
    __shared__ float sval[THREADS * V];
    const int lanes = 1 << S.lg, n_groups = THREADS >> S.lg;
    const int g = threadIdx.x >> S.lg;
    const int64_t row = blockIdx.x, j = threadIdx.x & (lanes - 1);
    const bool col_ok = j * V < S.D;
    const int64_t c = col_ok ? vec_col<V>(j, S.D) : 0;
    const float* __restrict__ part = S.partial + c;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    int any = 0;
    constexpr int U = 4;
    for (int t0 = g; t0 < tiles; t0 += U * n_groups) {
        uint32_t k[U];
        float f[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t0 + u * n_groups;
            const int64_t at = min(t, tiles - 1);
            const uint32_t m = met[S.by_row ? row * tiles + at : at * S.rows + row];
            k[u] = t < tiles ? m : 0u;
        }
        // (where a tile has no such run, what lies there is read and not used)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = min(t0 + u * n_groups, tiles - 1);
            const int64_t slot = S.by_row ? row * tiles + at : at * tile_runs(S.rows) + (k[u] ? k[u] - 1 : 0u);
#pragma unroll
            for (int i = 0; i < V; ++i) f[u][i] = part[slot * S.D + i];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += k[u] ? f[u][i] : 0.f;
            any |= k[u] != 0;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sval[i * THREADS + threadIdx.x] = acc[i];
    any = __syncthreads_or(any);
    for (int s = n_groups >> 1; s > 0; s >>= 1) {
        if (g < s) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                acc[i] += sval[i * THREADS + threadIdx.x + (s << S.lg)];
                sval[i * THREADS + threadIdx.x] = acc[i];
            }
        }
        __syncthreads();
    }
    if (g == 0 && col_ok) write_scaled<O, V>(out + row * S.D + c, acc, S.scale);
    if (threadIdx.x == 0 && S.touched && (any || !keep_touched)) S.touched[row] = any != 0;
}

namespace {

// clearing in a launch of its own: 64 KB per workgroup, eight workgroups per CU at most
int clear_grid(const Fill& F) { return (int)std::min<int64_t>(2048, (F.bytes + F.n_touched + 65535) / 65536); }

int ceil_log2(int64_t x) { int l = 0; while (((int64_t)1 << l) < x) ++l; return l; }

// How the gradient is cut up: by the numbers of ids, rows and columns and the vector width alone.
struct SegmentPlan { bool few, by_row; int vec, lg, per_group, pieces, segments; };
SegmentPlan plan_segments(int64_t N, int64_t rows, int64_t D, int type) {
    SegmentPlan p{};
    const int full = type == ELEM_F32 ? 4 : 8;
    p.vec = D >= full ? full : 1;
    const int64_t vectors = (D + p.vec - 1) / p.vec;
    p.lg = vectors >= 64 ? 6 : ceil_log2(vectors);
    p.segments = (int)((vectors + (1 << p.lg) - 1) >> p.lg);
    // few rows: a lane group of the tile sums at most 64 positions, the tiles' tables of the rows
    // they met stay below 16 MB, and what the two launches move for their split costs less than
    // the sorted form's passes.  They write and read the partial rows (as many as a tile has ids,
    // at most), and the join of more than 256 rows picks two bytes out of a line for every tile
    // and row; a pass costs what moving 64 MB and 90 bytes an id does.  Measured at 1 M ids, few
    // against sorted: 1000 rows of 12 float32 46 and 69 us, of 32 60 and 69; 2000 rows of 32 72
    // and 70, 4000 rows 90 and 69; 200 rows of 64 78 and 77, 500 rows 97 and 94, 2000 153 and 96.
    // At 250 k ids 4000 rows of 64 take 46 and 49 us
    const int64_t tiles = (N + kTileIds - 1) / kTileIds;
    p.by_row = rows <= 256;
    const int64_t passes = rows < kRadix ? 1 : 2;
    const int64_t split = 2 * tiles * tile_runs(rows) * D * 4 + (p.by_row ? 0 : 64 * tiles * rows);
    p.few = rows <= kFewRows && vectors <= 16 && tiles <= kFewTiles && tiles * rows <= (1 << 23) &&
            split <= passes * ((64 << 20) + 90 * N);
    if (p.few) {
        const int groups = kTileThreads >> p.lg;
        p.per_group = (int)((std::min<int64_t>(N, kTileIds) + groups - 1) / groups);
        p.pieces = (int)tiles;
        return p;
    }
    p.by_row = false;
    const int groups = 256 >> p.lg;
    // about 2048 workgroups (eight per CU) where there are enough ids; 4 positions at least (the
    // loads a lane keeps in flight), 64 at most (what one float32 sum may run over)
    const int64_t per = N * p.segments / ((int64_t)groups * 2048);
    p.per_group = 4;
    while (p.per_group < per && p.per_group < 64 && groups * p.per_group < kPieceMax) p.per_group *= 2;
    // (a few ids more per group spare the join)
    while (p.per_group < 16 && groups * p.per_group < N && groups * 16 >= N &&
           groups * p.per_group < kPieceMax) p.per_group *= 2;
    const int piece = groups * p.per_group;
    p.pieces = (int)((N + piece - 1) / piece);
    return p;
}

struct GradWorkspace {
    uint32_t *key[2], *val[2], *thist, *totals;
    float* partial;
    uint16_t* met;
    size_t bytes;
};
GradWorkspace carve_grad(void* ws, const SegmentPlan& s, int64_t N, int64_t rows, int64_t D) {
    GradWorkspace w;
    char* p = (char*)ws;
    size_t off = 0;
    auto take = [&](size_t bytes) { char* q = p + off; off += align256(bytes); return q; };
    const bool tiles = !s.few && N > kMergeSortMax;
    for (int i = 0; i < 2; ++i) {
        const bool need = !s.few && (i == 0 || N > kRun);
        w.key[i] = (uint32_t*)take(need ? 4 * (size_t)N : 0);
        w.val[i] = (uint32_t*)take(need ? 4 * (size_t)N : 0);
    }
    const size_t ntiles = ((size_t)N + kSortTile - 1) / kSortTile;
    w.thist = (uint32_t*)take(tiles ? 4 * kRadix * ntiles : 0);
    w.totals = (uint32_t*)take(tiles ? 4 * kRadix : 0);
    const size_t pieces = s.pieces > 1 ? s.pieces : 0;
    w.partial = (float*)take(sizeof(float) * pieces * (s.by_row ? rows : s.few ? tile_runs(rows) : 2) * D);
    w.met = (uint16_t*)take(s.few ? 2 * pieces * rows : 0);
    w.bytes = off;
    return w;
}

// Leaves the sorted pairs in key[*at], val[*at].
template <typename I>
int sort_runs(const I* ids, int N, IdRange range, int bits, const GradWorkspace& w, const Fill& F, int* at,
              hipStream_t s) {
    const int runs = cdiv(N, kRun);
    // clearing in 64 KB per workgroup, four per CU at most; three quarters beside the first
    // launch, which leaves more of every CU free, all of it where the merge takes most of the LDS
    auto blocks = [](const Fill& f) {
        return (int)std::min<int64_t>(1024, (f.bytes + f.n_touched + 65535) / 65536);
    };
    Fill A = F, B = F;
    if (runs > 1) {
        A.bytes = runs > 16 ? F.bytes : (F.bytes / 4 * 3) & ~(int64_t)15;
        A.n_touched = 0;
        B.rows = (char*)F.rows + A.bytes;
        B.bytes = F.bytes - A.bytes;
    }
    row_sort_runs_kernel<I><<<runs + blocks(A), 1024, 0, s>>>(ids, N, runs, range, bits, w.key[0], w.val[0], A);
    VINGS_LAUNCH_CHECK();
    *at = 0;
    if (runs == 1) return VINGS_OK;
    const int merge = cdiv(N, kMergeThreads);
    auto launch = [&](auto kernel) {
        kernel<<<merge + blocks(B), kMergeThreads, 0, s>>>(w.key[0], w.val[0], N, runs, merge, w.key[1], w.val[1], B);
    };
    if (runs <= 8) launch(row_merge_runs_kernel<8>);
    else if (runs <= 16) launch(row_merge_runs_kernel<16>);
    else launch(row_merge_runs_kernel<32>);
    VINGS_LAUNCH_CHECK();
    *at = 1;
    return VINGS_OK;
}

// Leaves the sorted pairs in key[*at], val[*at].
template <typename I, bool DIRECT>
int sort_tiles(const I* ids, int64_t N, IdRange range, int bits, const GradWorkspace& w, const Fill& F, int* at,
               hipStream_t s) {
    const int ntiles = cdiv(N, kSortTile);
    int cur = 1;
    for (int shift = 0; shift < bits; shift += kRadixBits) {
        const int nbits = std::min(kRadixBits, bits - shift);
        if (shift == 0)
            row_first_hist_kernel<I, DIRECT><<<ntiles + clear_grid(F), kSortThreads, 0, s>>>(ids, N, ntiles, w.thist,
                                                                                             range, F);
        else
            sort_tile_hist_kernel<uint32_t, DIRECT><<<ntiles, kSortThreads, 0, s>>>(w.key[cur], N, shift, ntiles,
                                                                                    w.thist, nullptr, range);
        VINGS_LAUNCH_CHECK();
        if (!DIRECT) {
            sort_scan_kernel<<<kRadix, 256, 0, s>>>(w.thist, ntiles, w.totals);
            VINGS_LAUNCH_CHECK();
        }
        if (shift == 0)
            sort_scatter_kernel<I, DIRECT><<<ntiles, kSortThreads, 0, s>>>(
                ids, nullptr, w.key[cur ^ 1], w.val[cur ^ 1], N, 0, ntiles, w.thist, w.totals, nullptr, nbits, range);
        else
            sort_scatter_kernel<uint32_t, DIRECT><<<ntiles, kSortThreads, 0, s>>>(
                w.key[cur], w.val[cur], w.key[cur ^ 1], w.val[cur ^ 1], N, shift, ntiles, w.thist, w.totals, nullptr,
                nbits, range);
        VINGS_LAUNCH_CHECK();
        cur ^= 1;
    }
    *at = cur;
    return VINGS_OK;
}

template <typename I>
int sort_ids(const I* ids, int64_t N, IdRange range, int bits, const GradWorkspace& w, const Fill& F, int* at,
             hipStream_t s) {
    if (N <= kMergeSortMax) return sort_runs<I>(ids, (int)N, range, bits, w, F, at, s);
    return N <= (int64_t)kDirectTiles * kSortTile ? sort_tiles<I, true>(ids, N, range, bits, w, F, at, s)
                                                  : sort_tiles<I, false>(ids, N, range, bits, w, F, at, s);
}

template <typename T, typename O, int V>
int segment_launches(const Segments& S, const SegmentPlan& p, const void* grad, void* out, hipStream_t s) {
    row_segment_kernel<T, O, V><<<dim3(p.pieces, p.segments), 256, 4 * (2 * ((256 >> p.lg) * p.per_group) + 2), s>>>(S, (const T*)grad, (O*)out);
    VINGS_LAUNCH_CHECK();
    if (p.pieces > 1) {
        row_join_kernel<O, V><<<dim3(p.pieces - 1, p.segments), 256, 0, s>>>(S, (O*)out, p.pieces);
        VINGS_LAUNCH_CHECK();
    }
    return VINGS_OK;
}

template <typename T, typename O, typename I, int V>
int few_launches(const Segments& S, const SegmentPlan& p, const GradWorkspace& w, const void* grad, const void* ids,
                 IdRange range, int bits, void* out, int keep_touched, hipStream_t s) {
    if (p.pieces == 1)
        row_tile_kernel<T, O, I, V, true><<<1, kTileThreads, 0, s>>>(S, (const T*)grad, (const I*)ids, range, bits, (O*)out, w.met,
                                                            keep_touched);
    else
        row_tile_kernel<T, O, I, V, false><<<p.pieces, kTileThreads, 0, s>>>(S, (const T*)grad, (const I*)ids, range, bits, (O*)out,
                                                                    w.met, keep_touched);
    VINGS_LAUNCH_CHECK();
    if (p.pieces > 1) {
        if (S.rows <= 512)
            row_tile_join_kernel<O, V, 1024><<<(int)S.rows, 1024, 0, s>>>(S, w.met, p.pieces, (O*)out, keep_touched);
        else
            row_tile_join_kernel<O, V, 256><<<(int)S.rows, 256, 0, s>>>(S, w.met, p.pieces, (O*)out, keep_touched);
        VINGS_LAUNCH_CHECK();
    }
    return VINGS_OK;
}

template <typename T, typename O>
int few_by_kind(const Segments& S, const SegmentPlan& p, const GradWorkspace& w, const void* grad, const void* ids,
                int id_bytes, IdRange range, int bits, void* out, int keep, hipStream_t s) {
    constexpr int V = Elem<T>::kVec;
    if (id_bytes == 8)
        return p.vec == 1 ? few_launches<T, O, int64_t, 1>(S, p, w, grad, ids, range, bits, out, keep, s)
                          : few_launches<T, O, int64_t, V>(S, p, w, grad, ids, range, bits, out, keep, s);
    return p.vec == 1 ? few_launches<T, O, int32_t, 1>(S, p, w, grad, ids, range, bits, out, keep, s)
                      : few_launches<T, O, int32_t, V>(S, p, w, grad, ids, range, bits, out, keep, s);
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
    VINGS_REQUIRE(N < ((int64_t)1 << 31) && V < ((int64_t)1 << 31) - 1 && D <= kMaxStride,
                  "ids and rows must fit 31 bits, columns 20");
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

extern "C" size_t vings_row_lookup_backward_workspace_bytes(int64_t n_ids, int64_t n_rows, int64_t n_cols,
                                                            int type) {
    const int64_t top = (int64_t)1 << 31;
    if (n_ids <= 0 || n_rows <= 0 || n_cols <= 0 || n_ids >= top || n_cols > kMaxStride || !elem_known(type)) return 0;
    return carve_grad(nullptr, plan_segments(n_ids, n_rows, n_cols, type), n_ids, n_rows, n_cols).bytes;
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
    ProfScope prof(PROF_AUX, s);
    if (n_ids == 0) {
        row_clear_kernel<<<clear_grid(F), 256, 0, s>>>(F);
        VINGS_LAUNCH_CHECK();
        return VINGS_OK;
    }
    VINGS_REQUIRE(grad && ids, "null pointer");
    VINGS_REQUIRE(grad_stride >= 0 && grad_stride <= kMaxStride, "gradient rows lie at most 2^20 elements apart");
    const auto apart = [&](const void* p, int64_t bytes) {     // ... from what the call writes
        const uintptr_t a = (uintptr_t)p, r = (uintptr_t)rows, t = (uintptr_t)touched;
        return (a + bytes <= r || r + F.bytes <= a) && (!touched || a + bytes <= t || t + n_rows <= a);
    };
    VINGS_REQUIRE(apart(grad, ((n_ids - 1) * grad_stride + n_cols) * elem_bytes(type)) && apart(ids, n_ids * id_bytes) &&
                      (!touched || (uintptr_t)touched + n_rows <= (uintptr_t)rows ||
                       (uintptr_t)rows + F.bytes <= (uintptr_t)touched),
                  "what is written overlaps another array of the call");
    VINGS_REQUIRE(((uintptr_t)grad & (elem_bytes(type) - 1)) == 0 && ((uintptr_t)ids & (id_bytes - 1)) == 0,
                  "element alignment");
    VINGS_REQUIRE(((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
    const SegmentPlan p = plan_segments(n_ids, n_rows, n_cols, type);
    const GradWorkspace w = carve_grad(workspace, p, n_ids, n_rows, n_cols);
    if (workspace_bytes < w.bytes) {
        set_error("row gradient workspace too small: %zu < %zu", workspace_bytes, w.bytes);
        return VINGS_ERR_CAPACITY;
    }
    VINGS_REQUIRE(workspace || w.bytes == 0, "null pointer");
    const IdRange range{(uint32_t)n_rows, padding_id};
    const int bits = std::max(1, bits_for((uint32_t)n_rows));
    Segments S{nullptr, nullptr, (int)n_ids, (uint32_t)n_rows, n_cols, grad_stride, p.lg, p.per_group, scale, touched,
               w.partial, p.by_row};
    if (p.few) {
        if (type == ELEM_F32) return few_by_kind<float, float>(S, p, w, grad, ids, id_bytes, range, bits, rows, keep_touched, s);
        if (type == ELEM_BF16)
            return rows_type == ELEM_F32
                ? few_by_kind<__bf16, float>(S, p, w, grad, ids, id_bytes, range, bits, rows, keep_touched, s)
                : few_by_kind<__bf16, __bf16>(S, p, w, grad, ids, id_bytes, range, bits, rows, keep_touched, s);
        return rows_type == ELEM_F32
            ? few_by_kind<_Float16, float>(S, p, w, grad, ids, id_bytes, range, bits, rows, keep_touched, s)
            : few_by_kind<_Float16, _Float16>(S, p, w, grad, ids, id_bytes, range, bits, rows, keep_touched, s);
    }
    int at = 0;
    const int rs = id_bytes == 8 ? sort_ids((const int64_t*)ids, n_ids, range, bits, w, F, &at, s)
                                 : sort_ids((const int32_t*)ids, n_ids, range, bits, w, F, &at, s);
    if (rs != VINGS_OK) return rs;
    VINGS_REQUIRE((256 >> p.lg) * p.per_group <= kPieceMax, "piece");
    S.keys = w.key[at];
    S.pos = w.val[at];
    if (type == ELEM_F32) return segment_by_width<float, float>(S, p, grad, rows, s);
    if (type == ELEM_BF16)
        return rows_type == ELEM_F32 ? segment_by_width<__bf16, float>(S, p, grad, rows, s)
                                     : segment_by_width<__bf16, __bf16>(S, p, grad, rows, s);
    return rows_type == ELEM_F32 ? segment_by_width<_Float16, float>(S, p, grad, rows, s)
                                 : segment_by_width<_Float16, _Float16>(S, p, grad, rows, s);
}
