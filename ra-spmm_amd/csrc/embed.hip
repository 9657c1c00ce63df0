// embed.hip — rows of a table by id times a factor, and the table's gradient.
//
//     out[i] = scale * table[ids[i]];  d_table[v] = scale * sum_{i: ids[i] = v} grad[i]
//
// Bound by memory: the lookup reads a table row and writes one for every position, the gradient
// reads a row for every position and writes every table row.  The gradient is a sum by sorted
// ids, so that its order is fixed and no two workgroups add to one row: (id, position) pairs are
// sorted with the positions of an id in ascending order, and every table row sums its run of
// them.  Ids that take no part (padding, or outside of the table) sort behind the last row.
//
// The sort goes by digits of up to 11 bits, lowest first, three launches a digit: counts of every
// workgroup's piece, their running sums for every digit, and the move, in which lanes of a wave
// with one digit find their order by ballots.  Up to 8,192 positions, one launch counts for each
// how many come before it (8,192: 11.6 us; the digits' six launches take 55 at 1e6).
//
// The sum takes equal runs of sorted positions, not of table rows, so that a row with most of the
// positions costs no more than others: a group of lanes adds its run's gradients and writes each
// table row that begins and ends there; what reaches over an edge is joined in LDS, and between
// workgroups by a second launch.  Table rows without positions are written by further workgroups
// of the first.
//
// Measured, lookup and gradient on the GPU: 1e6 positions on 1e6 rows of 256 in bf16 171 us (6.0 TB/s)
// and 221 (4.6 TB/s), the sort 55 and the join 9; 1e6 positions on 61 rows of 100 in fp16 44 and 58 (the
// gathers of 200 bytes take lines of 128: 5 TB/s of lines), 20 and 9; 8,192 positions on 200,000
// rows of 128 in fp32 4 and 20 (5.3 TB/s), 12 and 5.
#include <algorithm>
#include <type_traits>

#include "overlap.hpp"
#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxDim = 1 << 20;
constexpr int64_t kMaxCount = (int64_t(1) << 31) - (1 << 24);
constexpr int64_t kMaxBlocks = 1 << 20;
// An output past the last-level cache (256 MB) is written around the caches: lines that wait
// there to be written slow down what is read (rows of a small table to 384 MB: 102 us, around
// the caches 67); a smaller one, which the next kernel finds there, is not (192 MB: 30 us, 34).
// So is a gradient's: lookup and gradient of 1e6 positions on 1e6 rows of 256 in bf16 one after
// the other, 399 us, 382.
constexpr int64_t kAroundBytes = int64_t(256) << 20;
constexpr int kRowsAhead = 4;     // rows that a group of the lookup takes at once
constexpr int kDigitBits = 11;
constexpr int kPiece = 4096;      // pairs of a workgroup in the sort,
constexpr int kMaxPieces = 512;   // more where there would be over this many of them,
constexpr int kMostPiece = 32768; // up to as many: more pieces then
constexpr int kMoveThreads = 512;
constexpr int kCountThreads = 1024;
// Positions that are sorted by counting, which is one launch but takes n^2 comparisons.  The
// gradient of 1,025 positions on 200,000 rows 12.6 us (by digits 39), of 8,192 20 (50); on 2,000
// rows, one digit, 12.4 (26) and 21 (34).
constexpr int kRankMost = 8192;
// Workgroups of the sum, about as many as are resident: 1e6 positions, 61 rows of 100 in fp16, sum
// and join 75 us (2,048: 80, 4,096: 86, 8,192: 98), and a row in all of them is joined from as many.
constexpr int kTiles = 1536;

struct EmbedArgs {
    const void* ids;
    const void* from;  // the table, or the gradient of out
    void* to;          // out, or the gradient of the table
    int64_t count, rows, padding;
    int64_t ld;  // below 2^31 where there is a second row
    int32_t dim;
    bool ids64, has_padding;
    float scale;
};

__device__ __forceinline__ int64_t id_at(const EmbedArgs& a, int64_t i) {
    return a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : (int64_t)static_cast<const int32_t*>(a.ids)[i];
}
__device__ __forceinline__ bool is_padding(const EmbedArgs& a, int64_t id) { return a.has_padding && id == a.padding; }
// The row that a position takes part in, `rows` where it does not.
__device__ __forceinline__ uint32_t key_at(const EmbedArgs& a, int64_t i) {
    const int64_t id = id_at(a, i);
    return (uint64_t)id < (uint64_t)a.rows && !is_padding(a, id) ? (uint32_t)id : (uint32_t)a.rows;
}

// P elements as they lie in memory: 16 bytes, at any address.  The last packet of a row that is
// not made of whole ones ends with the row: what it shares with the one before is computed and
// written by both, the same bits.
template <typename T, int P>
struct Packet {
    typedef T vec __attribute__((ext_vector_type(P), aligned(sizeof(T))));
};

// A group of 2^shift lanes takes kAhead rows at once, a packet of each per lane.  The rows of a
// workgroup lie side by side: lines that two workgroups share go to memory in two parts.
template <typename T, int P, bool AROUND>
__global__ __launch_bounds__(kThreads) void embed_rows(const EmbedArgs a, const int shift) {
    using vec = typename Packet<T, P>::vec;
    constexpr int kAhead = kRowsAhead;
    const uint32_t lane = threadIdx.x & ((1 << shift) - 1), groups = kThreads >> shift, count = (uint32_t)a.count;
    for (uint64_t first = (uint64_t)blockIdx.x * groups * kAhead; first < count; first += (uint64_t)gridDim.x * groups * kAhead) {
        const uint32_t i0 = (uint32_t)first + (threadIdx.x >> shift);
        int64_t id[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) id[u] = id_at(a, min(i0 + u * groups, count - 1));
        const T* from[kAhead];
        float by[kAhead], add[kAhead];  // by * v + add: -0 leaves the product; without a row 0 * 0 + 0, or NaN for ids outside
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const bool padding = is_padding(a, id[u]), inside = !padding && (uint64_t)id[u] < (uint64_t)a.rows;
            from[u] = inside ? static_cast<const T*>(a.from) + (uint64_t)(uint32_t)id[u] * (uint32_t)a.ld : nullptr;
            by[u] = inside ? a.scale : 0.f;  // a scale that is not finite makes no padding of its own
            add[u] = inside ? -0.f : padding ? 0.f : __builtin_nanf("");
        }
        T* const to = static_cast<T*>(a.to) + (uint64_t)i0 * (uint32_t)a.dim;
        for (uint32_t d0 = lane * P; d0 < (uint32_t)a.dim; d0 += P << shift) {
            const uint32_t d = min(d0, (uint32_t)a.dim - P);
            vec v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                v[u] = *reinterpret_cast<const vec*>(from[u] ? from[u] + d : reinterpret_cast<const T*>(kZeroRun));
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
#pragma unroll
                for (int e = 0; e < P; ++e) v[u][e] = (T)fmaf(by[u], (float)v[u][e], add[u]);
                if (i0 + u * groups >= count) continue;
                vec* const at = reinterpret_cast<vec*>(to + (uint64_t)(u * groups) * (uint32_t)a.dim + d);
                if constexpr (AROUND) __builtin_nontemporal_store(v[u], at);
                else *at = v[u];
            }
        }
    }
}

// ------------------------------------------------------------ the sort by id
struct SortArgs {
    EmbedArgs e;
    const uint2* from;  // pairs (key, position); NULL: the ids as they come
    uint2* to;
    uint32_t* counts;   // [digits][pieces]
    uint32_t* totals;   // [digits]
    int32_t count, piece, pieces, shift, digits;
};

__device__ __forceinline__ uint2 pair_at(const SortArgs& a, int i) {
    return a.from ? a.from[i] : make_uint2(key_at(a.e, i), (uint32_t)i);
}

__global__ __launch_bounds__(kCountThreads) void sort_count(const SortArgs a) {
    extern __shared__ uint32_t counts[];
    for (int d = threadIdx.x; d < a.digits; d += kCountThreads) counts[d] = 0;
    __syncthreads();
    const int first = blockIdx.x * a.piece, end = min(a.count, first + a.piece);
    for (int i0 = first + threadIdx.x; i0 < end; i0 += 4 * kCountThreads) {
        uint32_t key[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + u * kCountThreads, end - 1);
            key[u] = a.from ? a.from[i].x : key_at(a.e, i);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * kCountThreads < end) atomicAdd(&counts[(key[u] >> a.shift) & (a.digits - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += kCountThreads) a.counts[(int64_t)d * a.pieces + blockIdx.x] = counts[d];
}

// A wave per digit: the pieces' counts to their sums before each piece.
__global__ __launch_bounds__(kThreads) void sort_offsets(const SortArgs a) {
    const int digit = blockIdx.x * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (digit >= a.digits) return;
    uint32_t* const counts = a.counts + (int64_t)digit * a.pieces;
    uint32_t before = 0;
    for (int p = 0; p < a.pieces; p += 64) {
        const uint32_t mine = p + lane < a.pieces ? counts[p + lane] : 0;
        uint32_t sum = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = __shfl_up(sum, o, 64);
            if (lane >= o) sum += x;
        }
        if (p + lane < a.pieces) counts[p + lane] = before + sum - mine;
        before += __shfl(sum, 63, 64);
    }
    if (lane == 0) a.totals[digit] = before;
}

__global__ __launch_bounds__(kMoveThreads) void sort_move(const SortArgs a) {
    constexpr int kMoveWaves = kMoveThreads / 64, kRounds = kPiece / kMoveThreads;
    extern __shared__ uint32_t lds[];  // [digits] first places, [waves] sums, then [waves][digits] places past them, 16 bits each
    uint32_t* const start = lds;
    uint32_t* const wave_sums = lds + a.digits;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t* const counts = lds + a.digits + kMoveWaves + wave * (a.digits / 2);  // two digits a word
    for (int d = threadIdx.x; d < kMoveWaves * a.digits / 2; d += kMoveThreads) lds[a.digits + kMoveWaves + d] = 0;
    // Sums of the totals before each digit: a run of digits per thread.
    const int run = (a.digits + kMoveThreads - 1) / kMoveThreads, d0 = threadIdx.x * run;
    uint32_t mine = 0;
    for (int k = 0; k < run; ++k) mine += d0 + k < a.digits ? a.totals[d0 + k] : 0;
    uint32_t sum = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(sum, o, 64);
        if (lane >= o) sum += x;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    uint32_t before = sum - mine;
    for (int w = 0; w < wave; ++w) before += wave_sums[w];
    for (int k = 0; k < run && d0 + k < a.digits; ++k) {
        start[d0 + k] = before + a.counts[(int64_t)(d0 + k) * a.pieces + blockIdx.x];
        before += a.totals[d0 + k];
    }
    // Every wave takes its part of the piece, in order.
    const int part = a.piece / kMoveWaves, first = blockIdx.x * a.piece + wave * part, end = min(a.count, first + part);
    uint2 pair[kRounds];  // of kRounds rounds of the wave, loaded at once; most pieces have no more
    auto load = [&](int i0) {
#pragma unroll
        for (int r = 0; r < kRounds; ++r) pair[r] = pair_at(a, min(i0 + r * 64 + lane, a.count - 1));
    };
    for (int i0 = first; i0 < end; i0 += 64 * kRounds) {
        load(i0);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const uint32_t digit = (pair[r].x >> a.shift) & (a.digits - 1);
            if (i0 + r * 64 + lane < end) atomicAdd(&counts[digit / 2], digit & 1 ? 0x10000u : 1u);
        }
    }
    __syncthreads();
    // Counts to places: those of the waves before.  A piece holds fewer than 2^16 pairs.
    for (int d = threadIdx.x; d < a.digits / 2; d += kMoveThreads) {
        uint32_t at = 0;
        for (int w = 0; w < kMoveWaves; ++w) {
            uint32_t& x = lds[a.digits + kMoveWaves + w * (a.digits / 2) + d];
            const uint32_t n = x;
            x = at;
            at += n;
        }
    }
    __syncthreads();
    volatile uint16_t* const place = reinterpret_cast<volatile uint16_t*>(counts);
    for (int i0 = first; i0 < end; i0 += 64 * kRounds) {
        if (part > 64 * kRounds) load(i0);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const bool there = i0 + r * 64 + lane < end;
            const uint32_t digit = (pair[r].x >> a.shift) & (a.digits - 1);
            uint64_t same = __ballot(there);  // the lanes with this lane's digit
            for (uint32_t bit = 1; bit < (uint32_t)a.digits; bit <<= 1) {
                const uint64_t set = __ballot(there && (digit & bit));
                same &= digit & bit ? set : ~set;
            }
            const int before_me = __popcll(same & ((uint64_t(1) << lane) - 1));
            if (there) {
                const uint32_t at = place[digit];
                __builtin_amdgcn_wave_barrier();
                if (before_me == 0) place[digit] = (uint16_t)(at + __popcll(same));
                __builtin_amdgcn_wave_barrier();
                a.to[start[digit] + at + before_me] = pair[r];
            }
        }
    }
}

// Few positions: how many come before each, 32 of them a workgroup.  Its waves' halves share
// the others, 32 at a time: keys of positions before these count where they are not above,
// later ones where they are below.
__global__ __launch_bounds__(1024) void sort_rank(const EmbedArgs a, uint2* __restrict__ to) {
    __shared__ __align__(16) uint32_t keys[kRankMost];
    __shared__ int counts[32][32];
    const int n = (int)a.count, lane = threadIdx.x & 31, half = threadIdx.x >> 5, halves = blockDim.x >> 5;
    const int all = (n + 31) / 32;
    for (int j = threadIdx.x; j < all * 32; j += blockDim.x) keys[j] = j < n ? key_at(a, j) : 0xFFFFFFFFu;
    __syncthreads();
    const int mine = blockIdx.x * 32 + lane;
    const uint32_t key = keys[mine];
    int before = 0;
    for (int c = half; c < all; c += halves) {
        if (c == (int)blockIdx.x) {
            for (int j = 0; j < 32; ++j) {
                const uint32_t k = keys[c * 32 + j];
                before += k < key || (k == key && j < lane);
            }
        } else {
            const uint32_t below = key + (c < (int)blockIdx.x);  // keys are below 2^31
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const uint4 k = *reinterpret_cast<const uint4*>(keys + c * 32 + j);
                before += (k.x < below) + (k.y < below) + (k.z < below) + (k.w < below);
            }
        }
    }
    counts[half][lane] = before;
    __syncthreads();
    if (half == 0 && mine < n) {
        for (int h = 1; h < halves; ++h) before += counts[h][lane];
        to[before] = make_uint2(key, (uint32_t)mine);
    }
}

// ------------------------------------------------------------ the sums
// The first sorted pair of [lo, hi) whose key is not below `key`.
__device__ __forceinline__ int lower_bound(const uint2* pairs, int lo, int hi, uint32_t key) {
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (pairs[mid].x < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

struct SumArgs {
    EmbedArgs e;
    const uint2* pairs;
    float *heads, *tails;  // [tiles][dim]: what a tile adds to a row of an earlier one, and leaves for later ones
    int32_t count, shift, per, tile, tiles;
};

// kThreads table rows from first_row on: zeros where no position names them.
template <typename T, int P>
__device__ __forceinline__ void zero_rows(const SumArgs& a, int64_t first_row, int* lds) {
    using vec = typename Packet<T, P>::vec;
    const int rows = (int)min((int64_t)kThreads, a.e.rows - first_row);
    if (threadIdx.x < 2) lds[threadIdx.x] = lower_bound(a.pairs, 0, a.count, (uint32_t)(first_row + (threadIdx.x ? rows : 0)));
    __syncthreads();
    const int lo = lds[0], hi = lds[1];
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        const uint32_t v = (uint32_t)first_row + threadIdx.x;
        const int at = lower_bound(a.pairs, lo, hi, v);
        lds[threadIdx.x] = at < hi && a.pairs[at].x == v;
    }
    __syncthreads();
    vec zero;
#pragma unroll
    for (int e = 0; e < P; ++e) zero[e] = (T)0.f;
    const int lane = threadIdx.x & ((1 << a.shift) - 1), groups = kThreads >> a.shift;
    for (int r = threadIdx.x >> a.shift; r < rows; r += groups) {
        if (lds[r]) continue;
        T* const to = static_cast<T*>(a.e.to) + (first_row + r) * a.e.dim;
        for (int d = lane * P; d < a.e.dim; d += P << a.shift) *reinterpret_cast<vec*>(to + min(d, a.e.dim - P)) = zero;
    }
    __syncthreads();
}

// blockIdx.x: a tile of sorted positions, or past those workgroups that clear table rows
// (of the first column block); blockIdx.y: a block of P << shift columns.  A group of
// 2^shift lanes takes `per` positions of the tile, a packet of columns per lane.
template <typename T, int P, bool AROUND>
__global__ __launch_bounds__(kThreads) void embed_sum(const SumArgs a) {
    using vec = typename Packet<T, P>::vec;
    constexpr int kAhead = 4;  // rows in flight
    __shared__ float edge[2][kThreads * P];  // heads and tails of the groups
    __shared__ int flags[kThreads];          // 1: has a head, 2: has a tail, 4: the head reaches past the group
    if ((int)blockIdx.x >= a.tiles) {
        if (blockIdx.y != 0) return;
        const int64_t step = (int64_t)(gridDim.x - a.tiles) * kThreads;
        for (int64_t row = (int64_t)(blockIdx.x - a.tiles) * kThreads; row < a.e.rows; row += step) zero_rows<T, P>(a, row, flags);
        return;
    }
    const int group = threadIdx.x >> a.shift, groups = kThreads >> a.shift, lane = threadIdx.x & ((1 << a.shift) - 1);
    const int d0 = (((int)blockIdx.y << a.shift) + lane) * P, d = min(d0, a.e.dim - P);  // this lane's columns
    const bool there = d0 < a.e.dim;
    const T* const from = static_cast<const T*>(a.e.from) + d;
    const uint32_t rows = (uint32_t)a.e.rows;
    const int first = (int)blockIdx.x * a.tile + group * a.per, end = min(a.count, first + a.per);
    float acc[P];
#pragma unroll
    for (int e = 0; e < P; ++e) acc[e] = 0.f;
    auto write = [&](uint32_t row, const float* f) {
        if (!there) return;
        vec v;
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = (T)(a.e.scale * f[e]);
        vec* const at = reinterpret_cast<vec*>(static_cast<T*>(a.e.to) + (int64_t)row * a.e.dim + d);
        if constexpr (AROUND) __builtin_nontemporal_store(v, at);
        else *at = v;
    };
    float* const head = edge[0] + threadIdx.x * P;
    float* const tail = edge[1] + threadIdx.x * P;
    int flag = 0;
    if (first < end) {
        uint32_t row = a.pairs[first].x;
        bool begun = first == 0 || a.pairs[first - 1].x != row;  // the run of `row` begins in this group
        uint2 next[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) next[u] = a.pairs[min(first + u, end - 1)];
        for (int e0 = first; e0 < end && row < rows; e0 += kAhead) {
            uint2 pair[kAhead];
            vec v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) pair[u] = next[u];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) v[u] = *reinterpret_cast<const vec*>(from + (uint64_t)pair[u].y * (uint32_t)a.e.ld);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) next[u] = a.pairs[min(e0 + kAhead + u, end - 1)];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (e0 + u >= end) continue;
                if (pair[u].x != row) {
                    if (begun) {
                        write(row, acc);
                    } else {
                        flag |= 1;
#pragma unroll
                        for (int e = 0; e < P; ++e) head[e] = acc[e];
                    }
                    row = pair[u].x;
                    begun = true;
#pragma unroll
                    for (int e = 0; e < P; ++e) acc[e] = 0.f;
                    if (row >= rows) break;  // positions that take no part are the last
                }
#pragma unroll
                for (int e = 0; e < P; ++e) acc[e] += (float)v[u][e];
            }
        }
        if (row < rows) {  // the last run
            const bool on = end < a.count && a.pairs[end].x == row;
            if (begun && !on) {
                write(row, acc);
            } else {
                flag |= begun ? 2 : on ? 5 : 1;
                float* const to = begun ? tail : head;
#pragma unroll
                for (int e = 0; e < P; ++e) to[e] = acc[e];
            }
        }
    }
    if (lane == 0) flags[group] = flag;
    __syncthreads();
    // What reaches over an edge: from the group where the run begins, and from the tile's edge.
    auto follow = [&](int g) {  // adds the heads from group g on; whether the run reaches past the tile
        for (; g < groups; ++g) {
            const float* const from_head = edge[0] + ((g << a.shift) + lane) * P;
#pragma unroll
            for (int e = 0; e < P; ++e) acc[e] += from_head[e];
            if (!(flags[g] & 4)) return false;
        }
        return true;
    };
    const int64_t part = (int64_t)blockIdx.x * a.e.dim + d;
    if (group == 0 && (flags[0] & 1)) {
#pragma unroll
        for (int e = 0; e < P; ++e) acc[e] = 0.f;
        follow(0);
        if (there) {
#pragma unroll
            for (int e = 0; e < P; ++e) a.heads[part + e] = acc[e];
        }
    }
    if (flag & 2) {
#pragma unroll
        for (int e = 0; e < P; ++e) acc[e] = tail[e];
        if (!follow(group + 1)) {
            write(a.pairs[end - 1].x, acc);
        } else if (there) {
#pragma unroll
            for (int e = 0; e < P; ++e) a.tails[part + e] = acc[e];
        }
    }
}

// Rows that reach over tiles: a workgroup per tile in which one begins, whose threads' slices
// take the later tiles' heads in turn.
template <typename T>
__global__ __launch_bounds__(kThreads) void embed_join(const SumArgs a, const int shift) {
    __shared__ float sums[kThreads];
    const int tile = blockIdx.x, first = tile * a.tile, end = first + a.tile;
    if (end >= a.count) return;
    const uint32_t row = a.pairs[end - 1].x, next = a.pairs[end].x, before = first > 0 ? a.pairs[first - 1].x : row + 1;
    if (row >= (uint32_t)a.e.rows || next != row || before == row) return;  // nothing begins here and reaches past
    // Its last tile: most rows end in the next one; else steps of 1, 2, 4 .. tiles, then halves.
    int lo = tile + 1, hi = a.tiles;  // the last tile is in [lo, hi)
    for (int step = 1; lo + step < hi; step *= 2) {
        if (a.pairs[(lo + step) * a.tile].x != row) {
            hi = lo + step;
            break;
        }
        lo += step;
    }
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.pairs[mid * a.tile].x == row) lo = mid;
        else hi = mid;
    }
    const int lane = threadIdx.x & ((1 << shift) - 1), slice = threadIdx.x >> shift, slices = kThreads >> shift;
    for (int d0 = (int)blockIdx.y << shift; d0 < a.e.dim; d0 += (int)gridDim.y << shift) {
        const int d = d0 + lane;
        float x = 0.f;
        if (d < a.e.dim) {
#pragma unroll 8
            for (int t = tile + 1 + slice; t <= lo; t += slices) x += a.heads[(int64_t)t * a.e.dim + d];
        }
        sums[threadIdx.x] = x;
        __syncthreads();
        if (slice == 0 && d < a.e.dim) {
            x = a.tails[(int64_t)tile * a.e.dim + d];
            for (int i = 0; i < slices; ++i) x += sums[(i << shift) + lane];
            static_cast<T*>(a.e.to)[(int64_t)row * a.e.dim + d] = (T)(a.e.scale * x);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------ host side
ra_status check(const ra_embed_shape* s) {
    if (!s) return fail(RA_ERR_INVALID_ARGUMENT, "embed: shape is NULL");
    if (s->dtype != RA_DTYPE_F32 && s->dtype != RA_DTYPE_F16 && s->dtype != RA_DTYPE_BF16)
        return fail(RA_ERR_INVALID_ARGUMENT, "embed: unknown dtype");
    if (s->count < 0 || s->rows < 0 || s->dim < 1) return fail(RA_ERR_INVALID_ARGUMENT, "embed: bad sizes");
    if (s->dim > kMaxDim) return fail(RA_ERR_UNSUPPORTED, "embed: dim is at most 2^20");
    if (s->count >= kMaxCount) return fail(RA_ERR_UNSUPPORTED, "embed: too many positions (below 2^31 - 2^24)");
    if (s->rows >= INT32_MAX - 1) return fail(RA_ERR_UNSUPPORTED, "embed: too many table rows (below 2^31 - 2)");
    return RA_OK;
}

ra_status check_stride(int64_t rows, int64_t ld) {
    if (rows > 1 && ld > INT32_MAX) return fail(RA_ERR_UNSUPPORTED, "embed: rows are at most 2^31 - 1 elements apart");
    return RA_OK;
}

EmbedArgs args_of(const ra_embed_shape& s, const void* ids, const void* from, void* to, int64_t ld) {
    EmbedArgs a{};
    a.ids = ids;
    a.from = from;
    a.to = to;
    a.count = s.count;
    a.rows = s.rows;
    a.padding = s.padding;
    a.ld = ld;
    a.dim = s.dim;
    a.ids64 = s.ids64 != 0;
    a.has_padding = s.has_padding != 0;
    a.scale = s.scale;
    return a;
}

// Digits, pieces and the workspace of the sort: pairs twice (once where it is by counting),
// counts, totals.
struct SortPlan {
    int bits, passes, digit_bits, piece, pieces;
    int64_t pairs_bytes, bytes;
};
SortPlan sort_plan(const ra_embed_shape& s) {
    SortPlan p{};
    p.pairs_bytes = (s.count * 8 + 255) / 256 * 256;
    p.bytes = p.pairs_bytes;
    if (s.count <= kRankMost) return p;
    for (int64_t x = s.rows; x; x >>= 1) ++p.bits;  // keys are 0 .. rows
    p.bits = std::max(p.bits, 2);
    p.passes = (p.bits + kDigitBits - 1) / kDigitBits;
    p.digit_bits = (p.bits + p.passes - 1) / p.passes;
    p.piece = kPiece;
    while ((s.count + p.piece - 1) / p.piece > kMaxPieces && p.piece < kMostPiece) p.piece *= 2;
    p.pieces = static_cast<int>((s.count + p.piece - 1) / p.piece);
    p.bytes = 2 * p.pairs_bytes + ((int64_t(1) << p.digit_bits) * (p.pieces + 1) * 4 + 255) / 256 * 256;
    return p;
}

// The sorted pairs, in the workspace.
const uint2* sort(const EmbedArgs& e, const SortPlan& p, char* work, hipStream_t st) {
    uint2* const half[2] = {reinterpret_cast<uint2*>(work), reinterpret_cast<uint2*>(work + p.pairs_bytes)};
    if (p.passes == 0) {
        sort_rank<<<static_cast<int>((e.count + 31) / 32), e.count > 1024 ? 1024 : 256, 0, st>>>(e, half[0]);
        return half[0];
    }
    SortArgs a{};
    a.e = e;
    a.count = static_cast<int32_t>(e.count);
    a.piece = p.piece;
    a.pieces = p.pieces;
    a.digits = 1 << p.digit_bits;
    a.counts = reinterpret_cast<uint32_t*>(work + 2 * p.pairs_bytes);
    a.totals = a.counts + (int64_t)a.digits * p.pieces;
    for (int pass = 0; pass < p.passes; ++pass) {
        a.to = half[pass & 1];
        a.shift = pass * p.digit_bits;
        sort_count<<<p.pieces, kCountThreads, a.digits * 4, st>>>(a);
        sort_offsets<<<(a.digits + kWaves - 1) / kWaves, kThreads, 0, st>>>(a);
        sort_move<<<p.pieces, kMoveThreads, a.digits * 4 + kMoveThreads / 64 * (4 + a.digits * 2), st>>>(a);
        a.from = a.to;
    }
    return a.from;
}

// Elements of a packet: 16 bytes, or one where a row has not as many.
int packet_of(const ra_embed_shape& s) {
    const int p = s.dtype == RA_DTYPE_F32 ? 4 : 8;
    return s.dim < p ? 1 : p;
}
// Lanes of a row: a power of two, a wave at most.
int shift_of(int dim, int p) {
    int shift = 0;
    while (shift < 6 && (p << shift) < dim) ++shift;
    return shift;
}

// How the sum is cut: groups of lanes with `per` positions, tiles of a workgroup, blocks of
// columns.
struct SumPlan {
    int shift, per, tile, tiles, blocks;
};
SumPlan sum_plan(const ra_embed_shape& s) {
    const int p = packet_of(s);
    SumPlan x{};
    x.shift = shift_of(s.dim, p);
    x.blocks = (s.dim + (p << x.shift) - 1) / (p << x.shift);
    const int64_t groups = kThreads >> x.shift, most = std::max(kTiles / x.blocks, 256);
    x.per = static_cast<int>(std::max<int64_t>(4, (s.count + groups * most - 1) / (groups * most)));
    x.per = (x.per + 3) / 4 * 4;
    x.tile = static_cast<int>(groups * x.per);
    x.tiles = static_cast<int>((s.count + x.tile - 1) / x.tile);
    return x;
}
template <typename F>
void by_packet(int32_t dtype, int p, F f) {
    auto of_type = [&](auto t) {
        if (p == 1) f(t, std::integral_constant<int, 1>());
        else f(t, std::integral_constant<int, 16 / sizeof(t)>());
    };
    if (dtype == RA_DTYPE_F32) of_type(float());
    else if (dtype == RA_DTYPE_F16) of_type(f16_t());
    else of_type(bf16_t());
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_embed(const ra_embed_shape* s, const void* d_ids, const void* d_table, void* d_out, ra_stream_t stream) {
    RA_TRY(ra::check(s));
    if (s->count == 0) return RA_OK;
    RA_TRY(ra::check_stride(s->rows, s->ld_table));
    if (!d_ids || !d_out || (s->rows && !d_table)) return fail(RA_ERR_INVALID_ARGUMENT, "embed: NULL tensor");
    if (s->rows > 1 && s->ld_table < s->dim) return fail(RA_ERR_INVALID_ARGUMENT, "embed: rows overlap (ld_table is too small)");
    const int64_t size = s->dtype == RA_DTYPE_F32 ? 4 : 2;
    RA_TRY(ra::refuse_overlap("embed", {ra::rows_of("out", d_out, s->count, s->dim, s->dim, size)},
                              {ra::rows_of("ids", d_ids, s->count, 1, 1, s->ids64 ? 8 : 4),
                               ra::rows_of("the table", d_table, s->rows, s->dim, s->ld_table, size)}));
    const ra::EmbedArgs a = ra::args_of(*s, d_ids, d_table, d_out, s->ld_table);
    const bool around = s->count * s->dim * (s->dtype == RA_DTYPE_F32 ? 4 : 2) > ra::kAroundBytes;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int p = ra::packet_of(*s), shift = ra::shift_of(s->dim, p);
    const int64_t rows = (int64_t)(ra::kThreads >> shift) * ra::kRowsAhead;
    const int blocks = static_cast<int>(std::min((s->count + rows - 1) / rows, ra::kMaxBlocks));
    ra::by_packet(s->dtype, p, [&](auto t, auto packet) {
        using T = decltype(t);
        if (around) ra::embed_rows<T, decltype(packet)::value, true><<<blocks, ra::kThreads, 0, st>>>(a, shift);
        else ra::embed_rows<T, decltype(packet)::value, false><<<blocks, ra::kThreads, 0, st>>>(a, shift);
    });
    RA_LAUNCH_CHECK("embed");
    return RA_OK;
}

ra_status ra_embed_workspace(const ra_embed_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "embed: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = 0;
    if (s->count == 0) return RA_OK;
    *bytes = ra::sort_plan(*s).bytes + (int64_t)2 * ra::sum_plan(*s).tiles * s->dim * (int64_t)sizeof(float);
    return RA_OK;
}

ra_status ra_embed_backward(const ra_embed_shape* s, const void* d_ids, const void* d_grad, void* d_dtable,
                            void* d_workspace, int64_t bytes, ra_stream_t stream) {
    int64_t need = 0;
    RA_TRY(ra_embed_workspace(s, &need));
    if (s->rows == 0) return RA_OK;
    RA_TRY(ra::check_stride(s->count, s->ld_grad));
    if (!d_dtable || (s->count && (!d_ids || !d_grad))) return fail(RA_ERR_INVALID_ARGUMENT, "embed: NULL tensor");
    if (s->count > 1 && s->ld_grad < s->dim) return fail(RA_ERR_INVALID_ARGUMENT, "embed: rows overlap (ld_grad is too small)");
    if (bytes < need || (need && !d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "embed: the workspace is too small");
    if (need && !ra::aligned16(d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "embed: the workspace must be 16-byte aligned");
    const int64_t size = s->dtype == RA_DTYPE_F32 ? 4 : 2;
    RA_TRY(ra::refuse_overlap("embed",
                              {ra::rows_of("the table's gradient", d_dtable, s->rows, s->dim, s->dim, size),
                               {"the workspace", d_workspace, static_cast<uint64_t>(need)}},
                              {ra::rows_of("ids", d_ids, s->count, 1, 1, s->ids64 ? 8 : 4),
                               ra::rows_of("grad", d_grad, s->count, s->dim, s->ld_grad, size)}));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra::EmbedArgs a = ra::args_of(*s, d_ids, d_grad, d_dtable, s->ld_grad);
    const ra::SumPlan plan = ra::sum_plan(*s);
    ra::SumArgs sum{};
    sum.e = a;
    sum.count = static_cast<int32_t>(s->count);
    sum.shift = plan.shift;
    sum.per = plan.per;
    sum.tile = plan.tile;
    sum.tiles = plan.tiles;
    if (s->count) {
        const ra::SortPlan sorted = ra::sort_plan(*s);
        sum.pairs = ra::sort(a, sorted, static_cast<char*>(d_workspace), st);
        RA_LAUNCH_CHECK("embed sort");
        sum.heads = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + sorted.bytes);
        sum.tails = sum.heads + (int64_t)plan.tiles * s->dim;
    }
    const int64_t clear = std::min<int64_t>((s->rows + ra::kThreads - 1) / ra::kThreads, std::max(256, 65536 / plan.blocks));
    const dim3 grid(static_cast<uint32_t>(plan.tiles + clear), plan.blocks);
    const bool around = s->rows * s->dim * (s->dtype == RA_DTYPE_F32 ? 4 : 2) > ra::kAroundBytes;
    ra::by_packet(s->dtype, ra::packet_of(*s), [&](auto t, auto packet) {
        using T = decltype(t);
        if (around) ra::embed_sum<T, decltype(packet)::value, true><<<grid, ra::kThreads, 0, st>>>(sum);
        else ra::embed_sum<T, decltype(packet)::value, false><<<grid, ra::kThreads, 0, st>>>(sum);
        if (plan.tiles > 1)
            ra::embed_join<decltype(t)><<<dim3(plan.tiles, std::min((s->dim + 31) / 32, 16)), ra::kThreads, 0, st>>>(
                sum, std::min(ra::shift_of(s->dim, 1), 5));
    });
    RA_LAUNCH_CHECK("embed_sum");
    return RA_OK;
}

}  // extern "C"
