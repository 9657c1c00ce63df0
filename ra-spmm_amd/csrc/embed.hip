// embed.hip — rows of a table by id times a factor, and the table's gradient.
//
//     out[i] = scale * table[ids[i]];  d_table[v] = scale * sum_{i: ids[i] = v} grad[i]
//
// The gradient is a sum by sorted ids, so that its order is fixed and no two workgroups
// add to one row: (id, position) pairs are sorted with the positions of an id in
// ascending order, and every table row sums its run of them.  Ids that take no part
// (padding, or outside of the table) sort behind the last row.
//
// The sort goes by digits of up to 11 bits, lowest first, three launches a digit: counts
// of every workgroup's piece, their running sums for every digit, and the move, in which
// lanes of a wave with one digit find their order by ballots.
#include <algorithm>
#include <type_traits>

#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxDim = 1 << 20;
constexpr int64_t kMaxCount = (int64_t(1) << 31) - (1 << 24);
constexpr int64_t kMaxBlocks = 1 << 16;
constexpr int kDigitBits = 11;
constexpr int kPiece = 4096;      // pairs of a workgroup in the sort, more where there would be over
constexpr int kMaxPieces = 512;   // this many of them

struct EmbedArgs {
    const void* ids;
    const void* from;  // the table, or the gradient of out
    void* to;          // out, or the gradient of the table
    int64_t count, rows, padding, ld;
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

template <typename T>
__global__ __launch_bounds__(kThreads) void embed_rows(const EmbedArgs a) {
    for (int64_t i = blockIdx.x * kWaves + (threadIdx.x >> 6); i < a.count; i += (int64_t)gridDim.x * kWaves) {
        const int64_t id = id_at(a, i);
        const bool padding = is_padding(a, id), inside = (uint64_t)id < (uint64_t)a.rows;
        const T* const from = static_cast<const T*>(a.from) + (inside && !padding ? id : 0) * a.ld;
        T* const to = static_cast<T*>(a.to) + i * a.dim;
        for (int d = threadIdx.x & 63; d < a.dim; d += 64)
            to[d] = (T)(padding ? 0.f : inside ? a.scale * (float)from[d] : __builtin_nanf(""));
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

__global__ __launch_bounds__(kThreads) void sort_count(const SortArgs a) {
    extern __shared__ uint32_t counts[];
    for (int d = threadIdx.x; d < a.digits; d += kThreads) counts[d] = 0;
    __syncthreads();
    const int first = blockIdx.x * a.piece, end = min(a.count, first + a.piece);
    for (int i = first + threadIdx.x; i < end; i += kThreads) {
        const uint32_t key = a.from ? a.from[i].x : key_at(a.e, i);
        atomicAdd(&counts[(key >> a.shift) & (a.digits - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += kThreads) a.counts[(int64_t)d * a.pieces + blockIdx.x] = counts[d];
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

__global__ __launch_bounds__(kThreads) void sort_move(const SortArgs a) {
    extern __shared__ uint32_t lds[];  // [waves][digits] places, then [digits] totals' sums, [waves]
    uint32_t* const start = lds + kWaves * a.digits;
    uint32_t* const wave_sums = start + a.digits;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    volatile uint32_t* const place = lds + wave * a.digits;
    for (int d = threadIdx.x; d < kWaves * a.digits; d += kThreads) lds[d] = 0;
    // Sums of the totals before each digit: a run of digits per thread.
    const int run = (a.digits + kThreads - 1) / kThreads, d0 = threadIdx.x * run;
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
        start[d0 + k] = before;
        before += a.totals[d0 + k];
    }
    // Every wave takes a quarter of the piece, in order.
    const int quarter = a.piece / kWaves, first = blockIdx.x * a.piece + wave * quarter, end = min(a.count, first + quarter);
    for (int i = first + lane; i < end; i += 64) atomicAdd(&lds[wave * a.digits + ((pair_at(a, i).x >> a.shift) & (a.digits - 1))], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += kThreads) {
        uint32_t at = start[d] + a.counts[(int64_t)d * a.pieces + blockIdx.x];
        for (int w = 0; w < kWaves; ++w) {
            const uint32_t n = lds[w * a.digits + d];
            lds[w * a.digits + d] = at;
            at += n;
        }
    }
    __syncthreads();
    for (int i0 = first; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const bool there = i < end;
        const uint2 pair = there ? pair_at(a, i) : make_uint2(0, 0);
        const uint32_t digit = (pair.x >> a.shift) & (a.digits - 1);
        uint64_t same = __ballot(there);  // the lanes with this lane's digit
        for (uint32_t bit = 1; bit < (uint32_t)a.digits; bit <<= 1) {
            const uint64_t set = __ballot(there && (digit & bit));
            same &= digit & bit ? set : ~set;
        }
        const int before_me = __popcll(same & ((uint64_t(1) << lane) - 1));
        if (there) {
            const uint32_t at = place[digit];
            __builtin_amdgcn_wave_barrier();
            if (before_me == 0) place[digit] = at + __popcll(same);
            __builtin_amdgcn_wave_barrier();
            a.to[at + before_me] = pair;
        }
    }
}

// The first sorted pair whose key is not below `key`.
__device__ __forceinline__ int lower_bound(const uint2* pairs, int count, uint32_t key) {
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pairs[mid].x < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void embed_grad(const EmbedArgs a, const uint2* __restrict__ pairs) {
    for (int64_t v = blockIdx.x * kWaves + (threadIdx.x >> 6); v < a.rows; v += (int64_t)gridDim.x * kWaves) {
        const int first = lower_bound(pairs, (int)a.count, (uint32_t)v), end = lower_bound(pairs, (int)a.count, (uint32_t)v + 1);
        for (int d = threadIdx.x & 63; d < a.dim; d += 64) {
            float s = 0.f;
            for (int e = first; e < end; ++e) s += (float)static_cast<const T*>(a.from)[pairs[e].y * a.ld + d];
            static_cast<T*>(a.to)[v * a.dim + d] = (T)(a.scale * s);
        }
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

// Digits, pieces and the workspace of the sort: pairs twice, counts, totals.
struct SortPlan {
    int bits, passes, digit_bits, piece, pieces;
    int64_t pairs_bytes, counts_bytes;
};
SortPlan sort_plan(const ra_embed_shape& s) {
    SortPlan p{};
    for (int64_t x = s.rows; x; x >>= 1) ++p.bits;  // keys are 0 .. rows
    p.bits = std::max(p.bits, 1);
    p.passes = (p.bits + kDigitBits - 1) / kDigitBits;
    p.digit_bits = (p.bits + p.passes - 1) / p.passes;
    p.piece = kPiece;
    while ((s.count + p.piece - 1) / p.piece > kMaxPieces) p.piece *= 2;
    p.pieces = static_cast<int>((s.count + p.piece - 1) / p.piece);
    p.pairs_bytes = (s.count * 8 + 255) / 256 * 256;
    p.counts_bytes = ((int64_t(1) << p.digit_bits) * (p.pieces + 1) * 4 + 255) / 256 * 256;
    return p;
}

// The sorted pairs, in one of the workspace's two halves.
const uint2* sort(const EmbedArgs& e, const SortPlan& p, char* work, hipStream_t st) {
    uint2* const half[2] = {reinterpret_cast<uint2*>(work), reinterpret_cast<uint2*>(work + p.pairs_bytes)};
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
        sort_count<<<p.pieces, kThreads, a.digits * 4, st>>>(a);
        sort_offsets<<<(a.digits + kWaves - 1) / kWaves, kThreads, 0, st>>>(a);
        sort_move<<<p.pieces, kThreads, (kWaves * a.digits + a.digits + kWaves) * 4, st>>>(a);
        a.from = a.to;
    }
    return a.from;
}

template <typename F>
void by_type(int32_t dtype, F f) {
    if (dtype == RA_DTYPE_F32) f(float());
    else if (dtype == RA_DTYPE_F16) f(f16_t());
    else f(bf16_t());
}

int blocks_of(int64_t rows) {
    return static_cast<int>(std::min((rows + kWaves - 1) / kWaves, kMaxBlocks));
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_embed(const ra_embed_shape* s, const void* d_ids, const void* d_table, void* d_out, ra_stream_t stream) {
    RA_TRY(ra::check(s));
    if (s->count == 0) return RA_OK;
    if (!d_ids || !d_out || (s->rows && !d_table)) return fail(RA_ERR_INVALID_ARGUMENT, "embed: NULL tensor");
    if (s->rows > 1 && s->ld_table < s->dim) return fail(RA_ERR_INVALID_ARGUMENT, "embed: rows overlap (ld_table is too small)");
    const ra::EmbedArgs a = ra::args_of(*s, d_ids, d_table, d_out, s->ld_table);
    ra::by_type(s->dtype, [&](auto t) {
        ra::embed_rows<decltype(t)><<<ra::blocks_of(s->count), ra::kThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
    });
    RA_LAUNCH_CHECK("embed");
    return RA_OK;
}

ra_status ra_embed_workspace(const ra_embed_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "embed: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = 0;
    if (s->count == 0) return RA_OK;
    const ra::SortPlan p = ra::sort_plan(*s);
    *bytes = 2 * p.pairs_bytes + p.counts_bytes;
    return RA_OK;
}

ra_status ra_embed_backward(const ra_embed_shape* s, const void* d_ids, const void* d_grad, void* d_dtable,
                            void* d_workspace, int64_t bytes, ra_stream_t stream) {
    int64_t need = 0;
    RA_TRY(ra_embed_workspace(s, &need));
    if (s->rows == 0) return RA_OK;
    if (!d_dtable || (s->count && (!d_ids || !d_grad))) return fail(RA_ERR_INVALID_ARGUMENT, "embed: NULL tensor");
    if (s->count > 1 && s->ld_grad < s->dim) return fail(RA_ERR_INVALID_ARGUMENT, "embed: rows overlap (ld_grad is too small)");
    if (bytes < need || (need && !d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "embed: the workspace is too small");
    if (need && !ra::aligned16(d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "embed: the workspace must be 16-byte aligned");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra::EmbedArgs a = ra::args_of(*s, d_ids, d_grad, d_dtable, s->ld_grad);
    const uint2* pairs = nullptr;
    if (s->count) {
        pairs = ra::sort(a, ra::sort_plan(*s), static_cast<char*>(d_workspace), st);
        RA_LAUNCH_CHECK("embed sort");
    }
    ra::by_type(s->dtype, [&](auto t) {
        ra::embed_grad<decltype(t)><<<ra::blocks_of(s->rows), ra::kThreads, 0, st>>>(a, pairs);
    });
    RA_LAUNCH_CHECK("embed_grad");
    return RA_OK;
}

}  // extern "C"
