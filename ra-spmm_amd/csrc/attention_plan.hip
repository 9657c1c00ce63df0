// attention_plan.hip — plan of the graph attention (pieces of rows, transposed
// lists) and the C entries that run it.
#include <hipcub/hipcub.hpp>

#include <algorithm>
#include <memory>
#include <new>
#include <string>

#include "attention.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;

unsigned blocks_for(int64_t n) { return static_cast<unsigned>((n + kThreads - 1) / kThreads); }

// What the host reads back.  bad: rowptr decreases or has wrong ends, or a column
// is out of range.
struct Totals {
    unsigned long long items_slots;  // items << 32 | slots
    int32_t splits;
    int32_t bad;
};

__global__ __launch_bounds__(kThreads) void check_columns(const int32_t* __restrict__ idx, int64_t n, int32_t K,
                                                          Totals* __restrict__ out) {
    const int64_t stride = (int64_t)gridDim.x * kThreads;
    bool bad = false;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += stride) bad |= (uint32_t)idx[i] >= (uint32_t)K;
    if (bad) out->bad = 1;
}

// Pieces, slots and cuts of every row; entry `rows` gets zeros, so that the
// exclusive sums end with the totals.
__global__ __launch_bounds__(kThreads) void count_pieces(const int32_t* __restrict__ ptr, int32_t rows, int64_t nnz,
                                                         unsigned long long* __restrict__ items_slots,
                                                         int32_t* __restrict__ splits, Totals* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i > rows) return;
    int64_t n = 0;
    if (i < rows) {
        n = (int64_t)ptr[i + 1] - ptr[i];
        if (n < 0 || (i == 0 && ptr[0] != 0) || (i == rows - 1 && ptr[rows] != nnz)) out->bad = 1;
        n = max(n, (int64_t)0);
    }
    const unsigned long long pieces = i == rows ? 0 : n == 0 ? 1 : (n + kAttnPiece - 1) / kAttnPiece;
    items_slots[i] = pieces << 32 | (pieces > 1 ? pieces : 0);
    splits[i] = pieces > 1;
}

__global__ __launch_bounds__(kThreads) void place_pieces(const int32_t* __restrict__ ptr, int32_t rows,
                                                         const unsigned long long* __restrict__ items_slots,
                                                         const int32_t* __restrict__ splits, int4* __restrict__ items,
                                                         int4* __restrict__ split_rows) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= rows) return;
    const int begin = ptr[i], end = ptr[i + 1];
    const int64_t item = items_slots[i] >> 32;
    const int slot = static_cast<int>(items_slots[i] & 0xFFFFFFFFu);
    const int pieces = static_cast<int>((items_slots[i + 1] >> 32) - item);
    if (pieces == 1) {
        items[item] = make_int4(static_cast<int>(i), begin, end, -1);
        return;
    }
    for (int k = 0; k < pieces; ++k) {
        const int64_t b = (int64_t)begin + (int64_t)k * kAttnPiece;
        items[item + k] = make_int4(static_cast<int>(i), static_cast<int>(b),
                                    static_cast<int>(min(b + kAttnPiece, (int64_t)end)), slot + k);
    }
    split_rows[splits[i]] = make_int4(static_cast<int>(i), slot, pieces, 0);
}

__global__ __launch_bounds__(kThreads) void read_totals(const unsigned long long* __restrict__ items_slots,
                                                        const int32_t* __restrict__ splits, int32_t rows,
                                                        Totals* __restrict__ out) {
    out->items_slots = items_slots[rows];
    out->splits = splits[rows];
}

__global__ __launch_bounds__(kThreads) void edge_numbers(int64_t n, int32_t* __restrict__ out) {
    const int64_t stride = (int64_t)gridDim.x * kThreads;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < n; e += stride) out[e] = static_cast<int32_t>(e);
}

// Row of every edge in CSR order, a wave for each piece.
__global__ __launch_bounds__(kThreads) void edge_rows(const int4* __restrict__ items, int32_t num_items,
                                                      int32_t* __restrict__ out) {
    const int64_t waves = (int64_t)gridDim.x * (kThreads / 64);
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 6; i < num_items; i += waves) {
        const int4 it = items[i];
        for (int64_t e = (int64_t)it.y + (threadIdx.x & 63); e < it.z; e += 64) out[e] = it.x;
    }
}

__global__ __launch_bounds__(kThreads) void transposed_rows(const int32_t* __restrict__ rows, int64_t n,
                                                            const int32_t* __restrict__ edge, int32_t* __restrict__ out) {
    const int64_t stride = (int64_t)gridDim.x * kThreads;
    for (int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x; t < n; t += stride) out[t] = rows[edge[t]];
}

// First sorted key that is at least i, for i = 0 .. K.
__global__ __launch_bounds__(kThreads) void transposed_ptr(const int32_t* __restrict__ keys, int64_t n, int32_t K,
                                                           int32_t* __restrict__ ptr) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i > K) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (keys[mid] < i) lo = mid + 1;
        else hi = mid;
    }
    ptr[i] = static_cast<int32_t>(lo);
}

// Pieces of one side.  `tot`: device totals, with the checks of the columns done.
ra_status cut(AttnSide& s, int64_t nnz, Totals* tot, hipStream_t st) {
    const int64_t n = (int64_t)s.rows + 1;
    DeviceBuffer work;
    size_t scan_a = 0, scan_b = 0;
    RA_HIP_TRY(hipcub::DeviceScan::ExclusiveSum(nullptr, scan_a, (unsigned long long*)nullptr, (unsigned long long*)nullptr,
                                                static_cast<int>(n), st));
    RA_HIP_TRY(hipcub::DeviceScan::ExclusiveSum(nullptr, scan_b, (int32_t*)nullptr, (int32_t*)nullptr, static_cast<int>(n), st));
    const size_t scan = (std::max(scan_a, scan_b) + 15) / 16 * 16;
    RA_TRY(work.allocate(scan + n * 12 + 16));
    void* tmp = work.get();
    auto* items_slots = reinterpret_cast<unsigned long long*>(work.get<char>() + scan);
    auto* splits = reinterpret_cast<int32_t*>(items_slots + n);
    count_pieces<<<blocks_for(n), kThreads, 0, st>>>(s.ptr, s.rows, nnz, items_slots, splits, tot);
    RA_LAUNCH_CHECK("count_pieces");
    RA_HIP_TRY(hipcub::DeviceScan::ExclusiveSum(tmp, scan_a, items_slots, items_slots, static_cast<int>(n), st));
    RA_HIP_TRY(hipcub::DeviceScan::ExclusiveSum(tmp, scan_b, splits, splits, static_cast<int>(n), st));
    read_totals<<<1, 1, 0, st>>>(items_slots, splits, s.rows, tot);
    RA_LAUNCH_CHECK("read_totals");
    Totals t;
    RA_HIP_TRY(hipMemcpyAsync(&t, tot, sizeof(t), hipMemcpyDeviceToHost, st));
    RA_HIP_TRY(hipStreamSynchronize(st));
    if (t.bad)
        return fail(RA_ERR_INVALID_ARGUMENT,
                    "attention plan: rowptr must run from 0 to nnz without decreasing, and colind lie in [0, K)");
    const int64_t items = static_cast<int64_t>(t.items_slots >> 32);
    if (items > INT32_MAX) return fail(RA_ERR_UNSUPPORTED, "attention plan: more than 2^31 - 1 pieces of rows");
    s.num_items = static_cast<int32_t>(items);
    s.num_slots = static_cast<int64_t>(t.items_slots & 0xFFFFFFFFu);
    s.num_splits = t.splits;
    RA_TRY(s.lists.allocate((items + s.num_splits) * sizeof(int4)));
    auto* list = s.lists.get<int4>();
    s.items = list;
    s.splits = list + items;
    place_pieces<<<blocks_for(s.rows), kThreads, 0, st>>>(s.ptr, s.rows, items_slots, splits, list, list + items);
    RA_LAUNCH_CHECK("place_pieces");
    RA_HIP_TRY(hipStreamSynchronize(st));
    work.reset_idle();
    return RA_OK;
}

ra_status transpose(ra_attn_plan* p, hipStream_t st) {
    const AttnSide& r = p->side[0];
    AttnSide& c = p->side[1];
    const int64_t nnz = p->info.nnz, K = p->info.K;
    c.rows = p->info.K;
    // ptr [K + 1], row [nnz], edge [nnz], each 16-byte aligned
    const int64_t a = (K + 4) / 4 * 4, b = (nnz + 3) / 4 * 4;
    RA_TRY(p->transposed.allocate((a + 2 * b) * sizeof(int32_t)));
    auto* ptr = p->transposed.get<int32_t>();
    int32_t *row = ptr + a, *edge = row + b;
    c.ptr = ptr;
    c.idx = row;
    c.edge = edge;
    DeviceBuffer work;
    int bits = 1;
    while (bits < 31 && (int64_t{1} << bits) < K) ++bits;
    size_t sort = 0;
    RA_HIP_TRY(hipcub::DeviceRadixSort::SortPairs(nullptr, sort, (const int32_t*)nullptr, (int32_t*)nullptr,
                                                  (const int32_t*)nullptr, (int32_t*)nullptr, static_cast<int>(nnz), 0,
                                                  bits, st));
    sort = (sort + 15) / 16 * 16;
    RA_TRY(work.allocate(sort + 2 * b * sizeof(int32_t)));
    auto* keys = reinterpret_cast<int32_t*>(work.get<char>() + sort);
    int32_t* numbers = keys + b;
    const unsigned grid = std::min(blocks_for(nnz), 65536u);
    if (nnz > 0) {
        edge_numbers<<<grid, kThreads, 0, st>>>(nnz, numbers);
        RA_LAUNCH_CHECK("edge_numbers");
        // Stable: a column's rows stay in ascending order.
        RA_HIP_TRY(hipcub::DeviceRadixSort::SortPairs(work.get(), sort, r.idx, keys, numbers, edge,
                                                      static_cast<int>(nnz), 0, bits, st));
        // The rows are written in order and gathered once; 0.49 ms at 23e6 edges, each found by bisection 1.25.
        edge_rows<<<std::min(blocks_for((int64_t)r.num_items * 64), 1u << 20), kThreads, 0, st>>>(r.items, r.num_items, numbers);
        RA_LAUNCH_CHECK("edge_rows");
        transposed_rows<<<grid, kThreads, 0, st>>>(numbers, nnz, edge, row);
        RA_LAUNCH_CHECK("transposed_rows");
    }
    transposed_ptr<<<blocks_for(K + 1), kThreads, 0, st>>>(keys, nnz, p->info.K, ptr);
    RA_LAUNCH_CHECK("transposed_ptr");
    RA_HIP_TRY(hipStreamSynchronize(st));
    work.reset_idle();
    return RA_OK;
}

ra_status build(ra_attn_plan* p, const int32_t* rowptr, const int32_t* colind, bool backward, hipStream_t st) {
    RA_HIP_TRY(hipGetDevice(&p->device));
    AttnSide& r = p->side[0];
    r.ptr = rowptr;
    r.idx = colind;
    r.rows = p->info.M;
    if (p->info.M > 0) {
        DeviceBuffer totals;
        RA_TRY(totals.allocate(sizeof(Totals)));
        auto* tot = totals.get<Totals>();
        const Totals zero{};
        RA_HIP_TRY(hipMemcpyAsync(tot, &zero, sizeof(zero), hipMemcpyHostToDevice, st));
        if (p->info.nnz > 0) {
            check_columns<<<std::min(blocks_for(p->info.nnz), 4096u), kThreads, 0, st>>>(colind, p->info.nnz, p->info.K, tot);
            RA_LAUNCH_CHECK("check_columns");
        }
        RA_TRY(cut(r, p->info.nnz, tot, st));
        if (backward && p->info.K > 0) {
            RA_TRY(transpose(p, st));
            RA_TRY(cut(p->side[1], p->info.nnz, tot, st));
        }
    } else if (backward && p->info.K > 0) {
        // No rows: the columns' lists are empty, their gradients zero.
        RA_TRY(transpose(p, st));
        DeviceBuffer totals;
        RA_TRY(totals.allocate(sizeof(Totals)));
        const Totals zero{};
        RA_HIP_TRY(hipMemcpyAsync(totals.get(), &zero, sizeof(zero), hipMemcpyHostToDevice, st));
        RA_TRY(cut(p->side[1], 0, totals.get<Totals>(), st));
    }
    const AttnSide& c = p->side[1];
    ra_attn_info& i = p->info;
    i.backward = backward;
    i.num_items = r.num_items;
    i.num_splits = r.num_splits;
    i.num_slots = r.num_slots;
    i.num_items_t = c.num_items;
    i.num_splits_t = c.num_splits;
    i.num_slots_t = c.num_slots;
    i.plan_bytes = (int64_t)(r.lists.bytes() + c.lists.bytes() + p->transposed.bytes());
    return RA_OK;
}

int log2_up(int64_t n) {
    int b = 0;
    while ((int64_t{1} << b) < n) ++b;
    return b;
}

AttnArgs args_of(const ra_attn_shape& s, const AttnLayout& l) {
    AttnArgs a{};
    a.q_heads = s.q_heads;
    a.kv_heads = s.kv_heads;
    a.group = s.q_heads / s.kv_heads;
    a.head_dim = s.head_dim;
    a.value_dim = s.value_dim;
    a.scale = s.scale;
    a.scale2 = s.scale * ra::kLog2e;
    a.ldq = s.ldq;
    a.ldk = s.ldk;
    a.ldv = s.ldv;
    const uint32_t size = s.dtype == RA_DTYPE_F32 ? 4 : 2;
    a.q_pitch = static_cast<uint32_t>(s.ldq) * size;
    a.k_pitch = static_cast<uint32_t>(s.ldk) * size;
    a.v_pitch = static_cast<uint32_t>(s.ldv) * size;
    a.g_pitch = static_cast<uint32_t>(s.q_heads * s.value_dim) * size;
    a.ragged = l.ragged;
    a.head_blocks = l.head_blocks;
    a.hb_shift = l.hb_shift;
    a.pieces = 1;
    return a;
}

// 32-bit offsets reach the gathered matrices: 24-bit factors, less than 4 GiB.
bool narrow(int64_t rows, std::initializer_list<uint32_t> pitches) {
    for (const uint32_t p : pitches)
        if (rows >= (1 << 24) || p >= (1u << 24) || rows * (int64_t)p >= (int64_t{1} << 32)) return false;
    return true;
}

void side_of(AttnArgs& a, const AttnSide& s, bool by_head) {
    a.items = s.items;
    a.ptr = s.ptr;
    a.idx = s.idx;
    a.edge = s.edge;
    a.rows = s.rows;
    a.num_units = static_cast<uint32_t>((int64_t)s.num_items * a.head_blocks);
    a.head_items = by_head ? s.num_items : 0;
}

// Pieces of every row of a plan-free call: about kAttnPiece edges, fewer where that
// leaves most of the GPU's wave slots empty, but at least 32.  The number goes by the
// mean: the rows' own lengths are not known on the host, and a row many times longer
// than the others has pieces as many times longer.
int plan_free_pieces(const ra_attn_shape& s, int32_t M, int64_t nnz) {
    if (M <= 0 || nnz <= 0) return 1;
    const int64_t mean = (nnz + M - 1) / M;
    const int64_t waves = (int64_t)M * s.q_heads;  // a wave holds one head or more
    int64_t piece = kAttnPiece;
    while (piece > 32 && waves * ((mean + piece - 1) / piece) < 2048) piece /= 2;
    return static_cast<int>(std::min<int64_t>((mean + piece - 1) / piece, 4096));
}

bool same_device(const ra_attn_plan* p) {
    int d = -1;
    return hipGetDevice(&d) == hipSuccess && d == p->device;
}

}  // namespace

// Waves that run at once: 4 for each of the 1024 SIMDs.  Below it one head a wave: 4 new rows of 6,000 edges,
// 8 heads: 9.7 us, 16.3 with all heads in a wave.
constexpr int64_t kFewWaves = 4096;

// Heads kept apart: every XCD works on the pieces of one part of the heads, so that
// its 4 MiB of L2 face that part of the gathered rows only.  It takes gathered rows
// past the L2s, a head's runs of whole 128-byte lines, and lists long enough that
// the larger number of waves does not matter.  Social graph of 50,000 rows of 80
// (heads of 32 + 32 and 64 in bf16, 51 MB): forward 385 against 492 us; community
// graph of 512,000 rows of 32: 2.09 against 1.18 ms.
bool attn_by_head(const ra_attn_shape& s, int64_t rows, int64_t gathered, int64_t nnz) {
    const int64_t size = s.dtype == RA_DTYPE_F32 ? 4 : 2;
    const int64_t key = 2 * s.head_dim * size, value = s.value_dim * size;
    return s.q_heads == s.kv_heads && s.kv_heads >= 2 && key % 128 == 0 && value % 128 == 0 && nnz >= 64 * rows &&
           gathered * s.kv_heads * (key + value) > (int64_t{32} << 20);
}

AttnLayout attn_layout(const ra_attn_shape& s, int heads, const AttnPtrs& p, int64_t pieces, bool by_head) {
    AttnLayout l{};
    l.lm = 1;
    while (l.lm * 8 < s.head_dim || l.lm * 16 < s.value_dim) l.lm *= 2;
    l.nv = s.value_dim <= 8 * l.lm ? 4 : 8;
    const int64_t size = s.dtype == RA_DTYPE_F32 ? 4 : 2;
    // Whole packets: every matrix' address, pitch and head width are multiples of them.
    auto whole = [&](int64_t key, int64_t value) {
        auto fits = [](const void* ptr, int64_t pitch, int64_t run, int64_t packet) {
            return reinterpret_cast<uintptr_t>(ptr) % packet == 0 && pitch % packet == 0 && run % packet == 0;
        };
        return fits(p.q, p.ldq * size, s.head_dim * size, key) && fits(p.k, p.ldk * size, s.head_dim * size, key) &&
               fits(p.v, p.ldv * size, s.value_dim * size, value) && fits(p.grad, p.ldg * size, s.value_dim * size, value);
    };
    l.packet = whole(16, std::min<int64_t>(16, l.nv * size)) ? 16 : whole(4, 4) ? 4 : 2;
    if (l.packet != 16) l.nv = 8;
    // Heads of a wave: as many as leave the fewest lanes without a head.
    const int most = log2_up(32 / l.lm);
    int best = 0;
    int64_t best_lanes = INT64_MAX;
    for (int b = most; b >= 0; --b) {
        const int64_t blocks = (heads + (1 << b) - 1) >> b;
        if ((blocks << b) < best_lanes) {
            best_lanes = blocks << b;
            best = b;
        }
    }
    // One head a wave where the launch would leave wave slots empty (kFewWaves), and
    // where heads are kept apart (attn_by_head).
    if (by_head) best = 0;
    while (best > 0 && pieces * ((heads + (1 << best) - 1) >> best) < kFewWaves) --best;
    l.hb_shift = best;
    l.head_blocks = (heads + (1 << best) - 1) >> best;
    l.ragged = s.head_dim != 8 * l.lm || s.value_dim != 2 * l.lm * l.nv || heads != l.head_blocks << best;
    return l;
}

ra_status attn_check(const ra_attn_shape* s, int32_t M, int32_t K) {
    if (!s) return fail(RA_ERR_INVALID_ARGUMENT, "attention: shape is NULL");
    if (s->dtype != RA_DTYPE_F32 && s->dtype != RA_DTYPE_F16 && s->dtype != RA_DTYPE_BF16)
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: unknown dtype");
    if (s->q_heads < 1 || s->kv_heads < 1 || s->q_heads % s->kv_heads != 0)
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: q_heads must be a positive multiple of kv_heads");
    if (s->head_dim < 1 || s->value_dim < 1) return fail(RA_ERR_INVALID_ARGUMENT, "attention: empty heads");
    if (s->head_dim > 128 || s->value_dim > 256 || s->q_heads > 1024)
        return fail(RA_ERR_UNSUPPORTED, "attention: head_dim is at most 128, value_dim at most 256, q_heads at most 1024");
    if (std::max({s->ldq, s->ldk, s->ldv}) >= int64_t{1} << 30)
        return fail(RA_ERR_UNSUPPORTED, "attention: rows lie at most 2^30 elements apart");
    if ((M > 0 && s->ldq < (int64_t)s->q_heads * 2 * s->head_dim) ||
        (K > 0 && (s->ldk < (int64_t)s->kv_heads * 2 * s->head_dim || s->ldv < (int64_t)s->kv_heads * s->value_dim)))
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: rows overlap (a leading dimension is too small)");
    return RA_OK;
}

}  // namespace ra

using ra::fail;

namespace {

// The pool's lists and the messages take host memory: no exception leaves a C entry.
template <typename F>
ra_status guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return RA_ERR_OUT_OF_MEMORY;
    }
}

ra_status check_output(const void* p, const char* what) {
    return ra::aligned16(p) ? RA_OK : fail(RA_ERR_INVALID_ARGUMENT, std::string("attention: ") + what + " is not 16-byte aligned");
}

}  // namespace

extern "C" {

ra_status ra_attn_plan_create(const int32_t* d_rowptr, const int32_t* d_colind, int32_t M, int32_t K, int64_t nnz,
                              int32_t backward, ra_stream_t stream, ra_attn_plan** out) {
    if (!out) return fail(RA_ERR_INVALID_ARGUMENT, "attention plan: out is NULL");
    *out = nullptr;
    if (M < 0 || K < 0 || nnz < 0) return fail(RA_ERR_INVALID_ARGUMENT, "attention plan: negative size");
    if (nnz > INT32_MAX || M == INT32_MAX || K == INT32_MAX)
        return fail(RA_ERR_UNSUPPORTED, "attention plan: int32 lists hold at most 2^31 - 1 edges");
    if ((M > 0 && !d_rowptr) || (nnz > 0 && !d_colind))
        return fail(RA_ERR_INVALID_ARGUMENT, "attention plan: NULL rowptr or colind");
    if (M == 0 && nnz > 0) return fail(RA_ERR_INVALID_ARGUMENT, "attention plan: edges without rows");
    std::unique_ptr<ra_attn_plan> p(new (std::nothrow) ra_attn_plan());
    if (!p) return fail(RA_ERR_OUT_OF_MEMORY, "attention plan allocation");
    p->info.M = M;
    p->info.K = K;
    p->info.nnz = nnz;
    RA_TRY(guarded([&] { return ra::build(p.get(), d_rowptr, d_colind, backward != 0, reinterpret_cast<hipStream_t>(stream)); }));
    *out = p.release();
    return RA_OK;
}

ra_status ra_attn_plan_get_info(const ra_attn_plan* p, ra_attn_info* info) {
    if (!p || !info) return fail(RA_ERR_INVALID_ARGUMENT, "attention plan info: NULL argument");
    *info = p->info;
    return RA_OK;
}

ra_status ra_attn_plan_export(const ra_attn_plan* p, const char* name, int32_t* dst, int64_t* count) {
    if (!p || !name || !count) return fail(RA_ERR_INVALID_ARGUMENT, "attention plan export: NULL argument");
    const std::string n(name);
    const ra::AttnSide &r = p->side[0], &c = p->side[1];
    const void* from = nullptr;
    int64_t k = 0;
    if (n == "items") { from = r.items; k = 4LL * r.num_items; }
    else if (n == "items_t") { from = c.items; k = 4LL * c.num_items; }
    else if (n == "splits") { from = r.splits; k = 4LL * r.num_splits; }
    else if (n == "splits_t") { from = c.splits; k = 4LL * c.num_splits; }
    else if (n == "rowptr_t") { from = c.ptr; k = c.ptr ? c.rows + 1LL : 0; }
    else if (n == "row_t") { from = c.idx; k = c.idx ? p->info.nnz : 0; }
    else if (n == "edge_t") { from = c.edge; k = c.edge ? p->info.nnz : 0; }
    else return fail(RA_ERR_INVALID_ARGUMENT, "attention plan export: unknown array '" + n + "'");
    *count = k;
    if (dst && k > 0) RA_HIP_TRY(hipMemcpy(dst, from, k * sizeof(int32_t), hipMemcpyDeviceToHost));
    return RA_OK;
}

void ra_attn_plan_destroy(ra_attn_plan* p) { delete p; }

ra_status ra_attn_plan_run(ra_attn_plan* p, const ra_attn_shape* shape, const void* d_q, const void* d_k,
                           const void* d_v, const float* d_lam, const float* d_bias, void* d_out, float* d_stats,
                           ra_stream_t stream) {
    if (!p) return fail(RA_ERR_INVALID_ARGUMENT, "attention: plan is NULL");
    RA_TRY(ra::attn_check(shape, p->info.M, p->info.K));
    if (p->info.M == 0) return RA_OK;
    if (!d_q || !d_lam || !d_out || (p->info.nnz > 0 && (!d_k || !d_v)))
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: NULL tensor");
    if (!ra::same_device(p)) return fail(RA_ERR_INVALID_ARGUMENT, "attention: the plan was built on another GPU");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra_attn_shape& s = *shape;
    const bool by_head = ra::attn_by_head(s, p->info.M, p->info.K, p->info.nnz);
    const ra::AttnLayout l = ra::attn_layout(
        s, s.q_heads, {d_q, d_k, d_v, d_out, s.ldq, s.ldk, s.ldv, (int64_t)s.q_heads * s.value_dim},
        p->side[0].num_items, by_head);
    RA_TRY(ra::attn_check_units(p->side[0].num_items, l));
    ra::AttnArgs a = ra::args_of(s, l);
    ra::side_of(a, p->side[0], by_head);
    a.wide = !ra::narrow(p->info.K, {a.k_pitch, a.v_pitch});
    RA_TRY(check_output(d_out, "out"));
    RA_TRY(check_output(d_stats, "stats"));
    RA_TRY(guarded([&] { return p->partial.ensure(p->side[0].num_slots * ra::attn_forward_slot(s) * sizeof(float), st); }));
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.lam = d_lam;
    a.bias = d_bias;
    a.out = d_out;
    a.stats = d_stats;
    a.partial = p->partial.get<float>();
    RA_TRY(ra::attn_forward_launch(s.dtype, l, a, st));
    return ra::attn_forward_join_launch(s.dtype, a, p->side[0].splits, p->side[0].num_splits, st);
}

ra_status ra_attn_plan_run_backward(ra_attn_plan* p, const ra_attn_shape* shape, const void* d_q, const void* d_k,
                                    const void* d_v, const float* d_lam, const float* d_bias, const float* d_stats,
                                    const void* d_grad_out, void* d_dq, void* d_dk, void* d_dv, float* d_dlam,
                                    ra_stream_t stream) {
    if (!p) return fail(RA_ERR_INVALID_ARGUMENT, "attention: plan is NULL");
    if (!p->info.backward)
        return fail(RA_ERR_INACTIVE_PLAN, "attention: the plan was built without the backward pass' lists");
    RA_TRY(ra::attn_check(shape, p->info.M, p->info.K));
    const int32_t M = p->info.M, K = p->info.K;
    if (!d_dlam || !d_lam || (M > 0 && (!d_q || !d_stats || !d_grad_out || !d_dq)) || (K > 0 && (!d_k || !d_v || !d_dk || !d_dv)))
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: NULL tensor");
    if (!ra::same_device(p)) return fail(RA_ERR_INVALID_ARGUMENT, "attention: the plan was built on another GPU");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra_attn_shape& s = *shape;
    const ra::AttnPtrs ptrs{d_q, d_k, d_v, d_grad_out, s.ldq, s.ldk, s.ldv, (int64_t)s.q_heads * s.value_dim};
    const ra::AttnSide &rows = p->side[0], &cols = p->side[1];
    const int64_t partial = std::max({rows.num_slots * ra::attn_row_slot(s), cols.num_slots * ra::attn_col_slot(s),
                                      (int64_t)2 * ra::kLamBlocks * s.q_heads});  // doubles
    RA_TRY(check_output(d_dq, "dq"));
    RA_TRY(check_output(d_dk, "dk"));
    RA_TRY(check_output(d_dv, "dv"));
    RA_TRY(check_output(d_stats, "stats"));
    const bool rows_by_head = ra::attn_by_head(s, M, K, p->info.nnz), cols_by_head = ra::attn_by_head(s, K, M, p->info.nnz);
    const ra::AttnLayout l = ra::attn_layout(s, s.q_heads, ptrs, rows.num_items, rows_by_head);
    const ra::AttnLayout lt = ra::attn_layout(s, s.kv_heads, ptrs, cols.num_items, cols_by_head);
    RA_TRY(ra::attn_check_units(rows.num_items, l));
    RA_TRY(ra::attn_check_units(cols.num_items, lt));
    RA_TRY(guarded([&] { return p->partial.ensure(partial * sizeof(float), st); }));
    RA_TRY(guarded([&] { return p->record.ensure((int64_t)M * s.q_heads * 2 * sizeof(float4), st); }));
    ra::AttnArgs a = ra::args_of(s, l);
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.grad = d_grad_out;
    a.lam = d_lam;
    a.bias = d_bias;
    a.stats = const_cast<float*>(d_stats);
    a.record = p->record.get<float4>();
    a.record_row = (cols_by_head ? 1 : s.q_heads) * 2 * sizeof(float4);
    a.record_head = (cols_by_head ? (int64_t)M : 1) * 2 * sizeof(float4);
    a.partial = p->partial.get<float>();
    a.rows = M;
    if (M > 0) {
        ra::side_of(a, rows, rows_by_head);
        a.wide = !ra::narrow(K, {a.k_pitch, a.v_pitch});
        a.out = d_dq;
        RA_TRY(ra::attn_rows_launch(s.dtype, l, a, st));
        RA_TRY(ra::attn_rows_join_launch(s.dtype, a, rows.splits, rows.num_splits, st));
    }
    RA_TRY(ra::attn_lam_launch(a, p->partial.get<double>(), d_dlam, st));
    if (K > 0) {
        a.head_blocks = lt.head_blocks;
        a.hb_shift = lt.hb_shift;
        a.ragged = lt.ragged;
        ra::side_of(a, cols, cols_by_head);
        a.wide = !ra::narrow(M, {a.q_pitch, a.g_pitch, static_cast<uint32_t>(s.q_heads * 2 * sizeof(float4))});
        a.out = d_dk;
        a.out2 = d_dv;
        RA_TRY(ra::attn_cols_launch(s.dtype, lt, a, st));
        RA_TRY(ra::attn_cols_join_launch(s.dtype, a, cols.splits, cols.num_splits, st));
    }
    return RA_OK;
}

ra_status ra_attn_csr_workspace(const ra_attn_shape* shape, int32_t M, int64_t nnz, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "attention: bytes is NULL");
    RA_TRY(ra::attn_check(shape, 0, 0));
    if (M < 0 || nnz < 0) return fail(RA_ERR_INVALID_ARGUMENT, "attention: negative size");
    const int pieces = ra::plan_free_pieces(*shape, M, nnz);
    *bytes = pieces == 1 ? 0 : (int64_t)M * pieces * ra::attn_forward_slot(*shape) * (int64_t)sizeof(float);
    return RA_OK;
}

ra_status ra_attn_csr(const int32_t* d_rowptr, const int32_t* d_colind, int32_t M, int32_t K, int64_t nnz,
                      const ra_attn_shape* shape, const void* d_q, const void* d_k, const void* d_v,
                      const float* d_lam, const float* d_bias, void* d_out, void* d_workspace, int64_t bytes,
                      ra_stream_t stream) {
    if (M < 0 || K < 0 || nnz < 0 || nnz > INT32_MAX) return fail(RA_ERR_INVALID_ARGUMENT, "attention: bad size");
    RA_TRY(ra::attn_check(shape, M, K));
    if (M == 0) return RA_OK;
    if (!d_rowptr || !d_q || !d_lam || !d_out || (nnz > 0 && (!d_colind || !d_k || !d_v)))
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: NULL tensor");
    int64_t need = 0;
    RA_TRY(ra_attn_csr_workspace(shape, M, nnz, &need));
    if (bytes < need || (need > 0 && (!d_workspace || !ra::aligned16(d_workspace))))
        return fail(RA_ERR_INVALID_ARGUMENT, "attention: the workspace is too small or not 16-byte aligned");
    RA_TRY(check_output(d_out, "out"));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra_attn_shape& s = *shape;
    const int pieces = ra::plan_free_pieces(s, M, nnz);
    const ra::AttnLayout l = ra::attn_layout(
        s, s.q_heads, {d_q, d_k, d_v, d_out, s.ldq, s.ldk, s.ldv, (int64_t)s.q_heads * s.value_dim}, (int64_t)M * pieces, false);
    ra::AttnArgs a = ra::args_of(s, l);
    a.ptr = d_rowptr;
    a.idx = d_colind;
    a.rows = M;
    a.pieces = pieces;
    const int64_t units = (int64_t)M * a.pieces * a.head_blocks;
    if (units > ra::kMostUnits) return fail(RA_ERR_UNSUPPORTED, "attention: too many rows and heads without a plan");
    a.num_units = static_cast<uint32_t>(units);
    a.wide = !ra::narrow(K, {a.k_pitch, a.v_pitch});
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.lam = d_lam;
    a.bias = d_bias;
    a.out = d_out;
    a.partial = static_cast<float*>(d_workspace);
    RA_TRY(ra::attn_forward_launch(s.dtype, l, a, st));
    return a.pieces == 1 ? RA_OK : ra::attn_forward_join_launch(s.dtype, a, nullptr, M, st);
}

}  // extern "C"
