// Stable least-significant-digit radix passes over 32-bit keys with a 32-bit value, 8 bits a
// pass, written for 64-lane wavefronts: per-tile digit histogram, scan of every digit's row,
// scatter through LDS.  Used by the tile binning (surfel_bin.hip: keys and values from arrays)
// and by the gradient of a row lookup (row_table.hip: the first pass reads the ids themselves,
// a value being the position of its id).
#pragma once
#include "common.hpp"

namespace vings {

constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;                        // keys per lane per tile
constexpr int kSortTile = kSortThreads * kSortItems;  // 2048 keys per workgroup
constexpr int kRadixBits = 8;
constexpr int kRadix = 1 << kRadixBits;

static inline int bits_for(uint32_t span) {   // bits needed to hold values 0..span
    int bits = 0;
    while (bits < 32 && ((uint64_t)1 << bits) <= (uint64_t)span) ++bits;
    return bits;
}

static inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Sort key of a signed id: itself inside [0, rows), `rows` (behind every row) for the ids that
// name none and for the padding id.  Keys that are already 32-bit keys pass unchanged.
struct IdRange { uint32_t rows; int64_t padding; };
template <typename K> inline constexpr bool kIds = false;
template <> inline constexpr bool kIds<int32_t> = true;
template <> inline constexpr bool kIds<int64_t> = true;
template <typename K>
__device__ __forceinline__ uint32_t sort_key(K k, const IdRange& range) {
    if constexpr (kIds<K>)
        return k < 0 || (int64_t)k >= (int64_t)range.rows || (int64_t)k == range.padding ? range.rows
                                                                                         : (uint32_t)k;
    else
        return k;
}

__device__ __forceinline__ uint32_t digit_of(uint32_t k, int shift) {
    return (k >> shift) & (kRadix - 1);
}

// Digit histogram of one tile in one pass: thist[digit][tile], as the scan takes it, or, for a
// scatter that forms its prefixes itself (DIRECT), thist[tile][digit].
template <typename K, bool DIRECT>
static __device__ __forceinline__ void sort_tile_hist(const K* __restrict__ keys, int64_t D, int shift, int ntiles,
                                                      uint32_t* __restrict__ thist, IdRange range) {
    __shared__ uint32_t h[kRadix];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kSortTile;
    // (unguarded loads: one inside a divergent branch is waited for where the branch ends)
    uint32_t key[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r)
        key[r] = base < D ? sort_key(keys[min(base + r * kSortThreads + threadIdx.x, D - 1)], range) : 0u;
#pragma unroll
    for (int r = 0; r < kSortItems; ++r)
        if (base + r * kSortThreads + threadIdx.x < D) atomicAdd(&h[digit_of(key[r], shift)], 1u);
    __syncthreads();
    thist[DIRECT ? (size_t)blockIdx.x * kRadix + threadIdx.x : (size_t)threadIdx.x * ntiles + blockIdx.x] =
        h[threadIdx.x];
}

template <typename K, bool DIRECT = false>
static __global__ __launch_bounds__(kSortThreads) void sort_tile_hist_kernel(
    const K* __restrict__ keys, int64_t D, int shift, int ntiles,
    uint32_t* __restrict__ thist, const uint32_t* __restrict__ tail, IdRange range) {
    if (tail) D = min(D, (int64_t)tail[2]);
    sort_tile_hist<K, DIRECT>(keys, D, shift, ntiles, thist, range);
}

// One 256-lane workgroup per digit: exclusive scan of that digit's row of thist (per sort
// tile: keys with this digit in earlier tiles) and the row total into totals[digit]; the
// scatter adds the number of keys with a smaller digit itself.  Each lane owns 8 consecutive
// entries, so rows of up to 2048 sort tiles (4 M keys) take one round.
constexpr int kScanItems = 8;
static __global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t* __restrict__ thist, int ntiles,
                                                        uint32_t* __restrict__ totals) {
    __shared__ uint32_t wtot[4];
    __shared__ uint32_t carry_s;
    const int digit = blockIdx.x;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (threadIdx.x == 0) carry_s = 0;
    __syncthreads();
    uint32_t* row = thist + (size_t)digit * ntiles;
    for (int t0 = 0; t0 < ntiles; t0 += 256 * kScanItems) {
        const int first = t0 + threadIdx.x * kScanItems;
        uint32_t v[kScanItems], sum = 0;
#pragma unroll
        for (int k = 0; k < kScanItems; ++k) {
            v[k] = first + k < ntiles ? row[first + k] : 0u;
            sum += v[k];
        }
        const uint32_t inc = wave_scan_incl(sum);
        if (lane == 63) wtot[w] = inc;
        __syncthreads();
        uint32_t run = carry_s + inc - sum;
        for (int k = 0; k < w; ++k) run += wtot[k];
#pragma unroll
        for (int k = 0; k < kScanItems; ++k) {
            if (first + k < ntiles) row[first + k] = run;
            run += v[k];
        }
        __syncthreads();
        if (threadIdx.x == 255) carry_s = run;
        __syncthreads();
    }
    if (threadIdx.x == 0) totals[digit] = carry_s;
}

// Stable scatter of one tile.  Keys are held in a wave-striped arrangement
// (item r of lane l of wave w sits at tile_base + w*512 + r*64 + l) so that
// walking r = 0..7 visits each wave's segment in memory order.  Within a
// round the rank of a key among equal digits is the number of lower lanes
// holding the same digit, found with one ballot per digit bit.
// DIRECT: no scan went before; a lane adds its digit's counts over the tiles itself, a kilobyte a
// tile out of the L2, which up to kDirectTiles tiles takes less than the scan's launch (20 tiles,
// two passes: 35 instead of 39 us in all; 128 tiles: 47 instead of 46).
constexpr int kDirectTiles = 64;
template <typename K, bool DIRECT = false>
static __global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(
    const K* __restrict__ keys_in, const uint32_t* __restrict__ vals_in,
    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out, int64_t D, int shift,
    int ntiles, const uint32_t* __restrict__ thist, const uint32_t* __restrict__ totals,
    const uint32_t* __restrict__ tail, int nbits, IdRange range) {
    // nbits: significant bits of this pass's digit (the last pass of a 13-bit tile number has 5:
    // the ballots of the bits above are all-zero and skipped)
    __shared__ uint32_t wcount[4][kRadix];  // per-wave digit counts, then prefixes
    if (tail) D = min(D, (int64_t)tail[2]);
    __shared__ uint32_t gbase[kRadix];
    __shared__ uint32_t tile_off[kRadix];
    __shared__ uint32_t wsum4[4];
    __shared__ uint32_t lkey[kSortTile];
    __shared__ uint32_t lval[kSortTile];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t wbase = (int64_t)blockIdx.x * kSortTile + w * (kSortItems * 64);
    uint32_t key[kSortItems];
    uint32_t val[kSortItems];
    uint32_t rank[kSortItems];
    // (unguarded loads, see above, under way while the digit bases are formed; a speculative
    // launch may have tiles behind the last key)
    if ((int64_t)blockIdx.x * kSortTile < D) {
#pragma unroll
        for (int r = 0; r < kSortItems; ++r) {
            const int64_t i = wbase + r * 64 + lane, at = min(i, D - 1);
            key[r] = sort_key(keys_in[at], range);
            if constexpr (kIds<K>) val[r] = (uint32_t)i;
            else val[r] = vals_in[at];
        }
    }
    for (int k = threadIdx.x; k < 4 * kRadix; k += kSortThreads) (&wcount[0][0])[k] = 0;
    // first output slot of digit d in this tile = keys with a smaller digit anywhere
    // (exclusive prefix of the 256 digit totals, one digit per lane) + keys with digit d in
    // earlier tiles
    uint32_t tot = 0, earlier = 0;
    if constexpr (DIRECT) {
        constexpr int U = 16;
        for (int t0 = 0; t0 < ntiles; t0 += U) {
            uint32_t c[U];
#pragma unroll
            for (int u = 0; u < U; ++u) c[u] = thist[(size_t)min(t0 + u, ntiles - 1) * kRadix + threadIdx.x];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                tot += t0 + u < ntiles ? c[u] : 0u;
                earlier += t0 + u < (int)blockIdx.x ? c[u] : 0u;
            }
        }
    } else {
        tot = totals[threadIdx.x];
        earlier = thist[(size_t)threadIdx.x * ntiles + blockIdx.x];
    }
    const uint32_t inc = wave_scan_incl(tot);
    if (lane == 63) wsum4[w] = inc;
    __syncthreads();
    uint32_t below = inc - tot;
    for (int k = 0; k < w; ++k) below += wsum4[k];
    gbase[threadIdx.x] = below + earlier;
    __syncthreads();

    const uint64_t lt_mask = lane == 0 ? 0ull : (~0ull >> (64 - lane));
    // which lanes hold the same digit: independent for the rounds, so their ballots overlap
    uint32_t peers_n[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const bool valid = wbase + r * 64 + lane < D;
        if (!valid) key[r] = ~0u;
        const uint32_t d = digit_of(key[r], shift);
        uint64_t peers = __ballot(valid);
#pragma unroll
        for (int b = 0; b < kRadixBits; ++b) {
            if (b < nbits) {
                const uint64_t m = __ballot((d >> b) & 1u);
                peers &= ((d >> b) & 1u) ? m : ~m;
            }
        }
        // all lanes in `peers` share digit d (invalid lanes excluded)
        rank[r] = __popcll(peers & lt_mask);
        peers_n[r] = valid ? __popcll(peers) : 0u;
    }
    // ... then the chain of per-wave digit counters
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t d = digit_of(key[r], shift);
        const uint32_t before = wcount[w][d];  // read before the leader updates it
        const bool leader = peers_n[r] && rank[r] == 0;
        rank[r] += before;
        __builtin_amdgcn_wave_barrier();
        if (leader) wcount[w][d] = before + peers_n[r];
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // per digit: exclusive prefix over the 4 waves; then the digit's first slot inside the tile
    // (exclusive prefix of the tile's digit counts over the 256 digits, one per lane)
    {
        const int d = threadIdx.x;
        uint32_t run = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t c = wcount[k][d];
            wcount[k][d] = run;
            run += c;
        }
        const uint32_t inc2 = wave_scan_incl(run);
        if (lane == 63) wsum4[w] = inc2;
        __syncthreads();
        uint32_t off = inc2 - run;
        for (int k = 0; k < w; ++k) off += wsum4[k];
        tile_off[d] = off;
        gbase[d] -= off;   // output slot of tile position p with digit d = gbase[d] + p (mod 2^32)
    }
    __syncthreads();
    // Sort the tile in LDS, then write it out in order: consecutive lanes then store to
    // consecutive addresses inside each digit's run (a wave's store touches the few runs it
    // spans instead of up to 64 scattered lines).
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const int64_t i = wbase + r * 64 + lane;
        if (i < D) {
            const uint32_t d = digit_of(key[r], shift);
            const uint32_t p = tile_off[d] + wcount[w][d] + rank[r];
            lkey[p] = key[r];
            lval[p] = val[r];
        }
    }
    __syncthreads();
    const int64_t tile_base = (int64_t)blockIdx.x * kSortTile;
    const uint32_t n_valid = (uint32_t)max((int64_t)0, min((int64_t)kSortTile, D - tile_base));
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t p = r * kSortThreads + threadIdx.x;
        if (p < n_valid) {
            const uint32_t k = lkey[p];
            const uint32_t dst = gbase[digit_of(k, shift)] + p;
            keys_out[dst] = k;
            vals_out[dst] = lval[p];
        }
    }
}

}  // namespace vings
