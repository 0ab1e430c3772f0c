/*
 * Embedding lookup with scaling, and the table's gradient by sorted tokens (include/eri_layers.h).
 */
#include "eri_layers_device.h"

namespace eri_layers {
namespace {

constexpr uint32_t kThreads = 256;

struct Ids {
    const void *p;
    uint32_t wide; // 64-bit ids
    __device__ __forceinline__ int64_t operator[](uint32_t t) const { return wide ? ((const int64_t *)p)[t] : ((const int32_t *)p)[t]; }
};

struct LookupArgs {
    Ids ids;
    const void *table;
    void *out;
    uint32_t tokens, vocab, dim;
    uint64_t table_stride, out_stride;
    float scale;
};

/* L lanes to a row, U rows at a time in each thread's registers.  Bound by HBM: 16384 rows of 4096 bf16 36-42 us, 4.3-5.0 TB/s; one
 * prompt of 77 x 768 2.6 us, a launch and two trips to memory (the id, then the row).  One, two or eight rows at a time are level
 * or slower (16384 x 768 8.8, 8.0 and 8.2 us for 7.7).  Stores past the caches take 32 us for 36, but the norm that reads the rows
 * next then waits for memory: 85 us for both, against 80. */
template <typename T, int L, int U, bool SHORT> __global__ __launch_bounds__(kThreads) void embedding_kernel(const LookupArgs a) {
    constexpr uint32_t kRows = kThreads / L;
    const uint32_t first = blockIdx.x * kRows * U + threadIdx.x / L, lane = threadIdx.x % L;
    const T *row[U];
    bool real[U]; // the table's first row stands in for ids outside it
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t t = first + u * kRows;
        const int64_t id = t < a.tokens ? a.ids[t] : -1;
        real[u] = (uint64_t)id < a.vocab;
        row[u] = (const T *)a.table + (real[u] ? id * a.table_stride : 0);
    }
    for (uint32_t col = lane * 8; col < a.dim; col += L * 8) {
        Raw<T> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) load8<SHORT>(r[u], row[u], col, a.dim);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t t = first + u * kRows;
            settle8<SHORT>(r[u], col, a.dim);
            float v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] = real[u] ? r[u].get(e) * a.scale : 0.0f;
            if (t < a.tokens) store8((T *)a.out + t * a.out_stride, col, a.dim, v);
        }
    }
}

template <typename T, int L, bool SHORT = false> void launch_lookup(const LookupArgs &a, uint32_t compute_units, hipStream_t s) {
    constexpr uint32_t kRows = kThreads / L;
    if (!SHORT && a.tokens / (kRows * 4) >= compute_units * 4) // four rows a thread where that still fills the chip
        hipLaunchKernelGGL((embedding_kernel<T, L, 4, false>), dim3((a.tokens + kRows * 4 - 1) / (kRows * 4)), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((embedding_kernel<T, L, 1, SHORT>), dim3((a.tokens + kRows - 1) / kRows), dim3(kThreads), 0, s, a);
}
template <typename T> void launch_lookup_of(const LookupArgs &a, uint32_t compute_units, hipStream_t s) {
    if (a.dim < 8) launch_lookup<T, 8, true>(a, compute_units, s);
    else if (a.dim <= 64) launch_lookup<T, 8>(a, compute_units, s);
    else if (a.dim <= 256) launch_lookup<T, 32>(a, compute_units, s);
    else if (a.dim <= 1024) launch_lookup<T, 128>(a, compute_units, s);
    else launch_lookup<T, 256>(a, compute_units, s);
}

// ---------------------------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------------------------

/*
 * Sorting: ids are dealt to K = 2^shift buckets by their low bits, a workgroup to a bucket.  It reads all ids, in order and
 * each wave its share of them, counts its own ones and keeps their tokens; then it writes the tokens of each of its ids, in
 * ascending order, to its part of the sorted list.  Where that part begins, it has counted too, as the number of tokens
 * in the buckets before it: no workgroup waits for another.  Between the two it writes the rows that no token names:
 * stores that nothing waits for.
 *
 * Summing: the runs of equal ids in the sorted list are cut into pieces of 2^log_piece tokens, and a wave sums the pieces that
 * begin in its step of half as many places, for L*8 columns: its loads go ahead through the list whatever the lengths of the
 * runs, and a wave has at most a piece and a step less one of tokens.  A run of one piece is written as it ends; the pieces
 * of longer ones are left in the workspace and summed in their order by a third kernel.
 *
 * What bounds it: HBM where the table is large (32768 x 4096 bf16 into 128000 rows: 170 us for 1 GB of zeros and the sort,
 * 83 for the sums, 7 for the long runs; 4.8 TB/s in all, what a copy of that size reaches), three launches and their trips to
 * memory where it is not (4095 x 1155 accumulated into fp32: 5.4 + 8.4 + 5 us for 22 MB).  With rows of up to 64 tokens summed in
 * the sorting workgroup the large case took 577 us: a bucket's rows wait for memory one after the other.
 */
constexpr uint32_t kWaves = 16;       // of a bucket's workgroup: one workgroup a compute unit
constexpr uint32_t kLocalMost = 1024; // ids of a bucket
constexpr uint32_t kOwnMost = 512;    // tokens of a bucket that a wave keeps from the first look to the second
constexpr uint32_t kLogPieceMost = 5;
constexpr uint32_t kListMost = (1 << kLogPieceMost) * 3 / 2; // places that a step and the piece that it ends with take

struct Place { // of the sorted list
    uint32_t token, id;
    uint32_t at, run; // place within the run of tokens with that id, and the run's length
};

struct GradArgs {
    Ids ids;
    const void *grad;
    void *out;
    Place *sorted;    // tokens places, of which the first *used are set
    uint32_t *used;
    float *partial;   // sums of pieces, padded floats each
    uint32_t tokens, vocab, dim, shift, locals, padded, tiles, log_piece;
    uint64_t grad_stride, out_stride;
    int64_t padding_id;
    float scale;
    uint32_t accumulate, out_bytes, lanes; // lanes to a row of zeros
    __device__ __forceinline__ bool counts(int64_t id) const { return (uint64_t)id < vocab && id != padding_id; }
};

/* Where the sum of the piece at place `start` goes, of a run with several.  The pieces of a run begin one length of a piece
 * apart, and the next such run begins more than that behind this one's beginning: of those that begin within one length
 * of places, one at most is a run's first and one at most is not. */
__device__ __forceinline__ uint64_t slot_of(uint32_t start, bool first, uint32_t log_piece) { return 2 * (uint64_t)(start >> log_piece) + first; }

__global__ __launch_bounds__(1024) void embedding_sort_kernel(const GradArgs a) {
    extern __shared__ uint32_t counts[]; // kWaves x locals: first counts, then where the wave's next token of that id goes
    __shared__ uint32_t starts[kLocalMost], lengths[kLocalMost], part[kWaves], before[kWaves];
    __shared__ uint32_t own_token[kWaves][kOwnMost];
    __shared__ uint16_t own_local[kWaves][kOwnMost];
    const uint32_t bucket = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, mask = (1u << a.shift) - 1;
    for (uint32_t i = threadIdx.x; i < kWaves * a.locals; i += 1024) counts[i] = 0;
    __syncthreads();

    // count, and keep the bucket's own tokens: the first kOwnMost that a wave finds in its share
    const uint32_t share = (a.tokens + kWaves * kWave - 1) / (kWaves * kWave) * kWave;
    const uint32_t from = wave * share, to = from + share < a.tokens ? from + share : a.tokens;
    uint32_t *mine = counts + wave * a.locals, lower = 0, found = 0;
    constexpr uint32_t kIds = 8; // of a lane, under way together
    for (uint32_t set = from; set < to; set += kIds * kWave) {
        int64_t ids[kIds];
#pragma unroll
        for (uint32_t k = 0; k < kIds; ++k) {
            const uint32_t t = set + k * kWave + lane;
            ids[k] = a.ids[t < to ? t : to - 1];
        }
#pragma unroll
        for (uint32_t k = 0; k < kIds; ++k) {
            const uint32_t t = set + k * kWave + lane, id = (uint32_t)ids[k], b = id & mask;
            const bool use = t < to && a.counts(ids[k]), own = use && b == bucket;
            lower += (uint32_t)__popcll(__ballot(use && b < bucket));
            const uint64_t all = __ballot(own);
            if (!all) continue;
            const uint32_t n = found + (uint32_t)__popcll(all & ((1ull << lane) - 1));
            if (own) atomicAdd(&mine[id >> a.shift], 1u);
            if (own && n < kOwnMost) own_token[wave][n] = t, own_local[wave][n] = (uint16_t)(id >> a.shift);
            found += (uint32_t)__popcll(all);
        }
    }
    if (lane == 0) before[wave] = lower;
    __syncthreads();

    // places: a thread to an id
    uint32_t total = 0, base = 0;
    for (uint32_t w = 0; w < kWaves; ++w) base += before[w];
    if (threadIdx.x < a.locals)
        for (uint32_t w = 0; w < kWaves; ++w) total += counts[w * a.locals + threadIdx.x];
    uint32_t upto = total;
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t v = __shfl_up(upto, d);
        if ((int)lane >= d) upto += v;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    uint32_t start = base + upto - total, all_mine = 0;
    for (uint32_t w = 0; w < wave; ++w) start += part[w];
    for (uint32_t w = 0; w < kWaves; ++w) all_mine += part[w];
    if (bucket == gridDim.x - 1 && threadIdx.x == 0) *a.used = base + all_mine;
    if (threadIdx.x < a.locals) {
        starts[threadIdx.x] = start;
        lengths[threadIdx.x] = total;
        for (uint32_t w = 0; w < kWaves; ++w) {
            uint32_t *c = &counts[w * a.locals + threadIdx.x];
            const uint32_t n = *c;
            *c = start;
            start += n;
        }
    }
    __syncthreads();

    // rows without a token
    if (!a.accumulate)
        for (uint32_t local = threadIdx.x / a.lanes; local < a.locals; local += 1024 / a.lanes) {
            const uint32_t id = local << a.shift | bucket;
            if (id >= a.vocab || lengths[local]) continue;
            char *row = (char *)a.out + id * a.out_stride * a.out_bytes;
            const uint64_t bytes = (uint64_t)a.dim * a.out_bytes;
            for (uint64_t at = threadIdx.x % a.lanes * 16ull; at < bytes; at += a.lanes * 16ull) {
                if (at + 16 <= bytes) *(u32x4_at2 *)(row + at) = u32x4{0, 0, 0, 0};
                else
                    for (uint64_t b = at; b < bytes; b += 2) *(uint16_t *)(row + b) = 0;
            }
        }

    // the list: each wave for its share; of several tokens in one step, an id at a time
    if (all_mine == 0) return;
    auto put = [&](bool own, uint32_t token, uint32_t local_of) {
        const uint32_t start_of = starts[own ? local_of : 0], run_of = lengths[own ? local_of : 0];
        for (uint64_t left = __ballot(own); left;) {
            const uint32_t local = (uint32_t)__builtin_amdgcn_readlane((int)local_of, __builtin_ctzll(left));
            const bool same = own && local_of == local;
            const uint64_t all = __ballot(same);
            uint32_t place = 0;
            if (lane == 0) place = atomicAdd(&mine[local], (uint32_t)__popcll(all));
            place = (uint32_t)__builtin_amdgcn_readfirstlane((int)place);
            if (same) {
                place += (uint32_t)__popcll(all & ((1ull << lane) - 1));
                a.sorted[place] = Place{token, local << a.shift | bucket, place - start_of, run_of};
            }
            left &= ~all;
        }
    };
    if (found <= kOwnMost) {
        for (uint32_t at = 0; at < found; at += kWave) {
            const bool own = at + lane < found;
            put(own, own ? own_token[wave][at + lane] : 0, own ? own_local[wave][at + lane] : 0);
        }
        return;
    }
    for (uint32_t set = from; set < to; set += kIds * kWave) { // more than that: a second look
        int64_t ids[kIds];
#pragma unroll
        for (uint32_t k = 0; k < kIds; ++k) {
            const uint32_t t = set + k * kWave + lane;
            ids[k] = a.ids[t < to ? t : to - 1];
        }
#pragma unroll 1
        for (uint32_t k = 0; k < kIds; ++k) {
            const uint32_t t = set + k * kWave + lane;
            put(t < to && a.counts(ids[k]) && ((uint32_t)ids[k] & mask) == bucket, t, (uint32_t)ids[k] >> a.shift);
        }
    }
}

template <bool SHORT, typename TO> __device__ __forceinline__ void finish8(const GradArgs &a, uint32_t id, uint32_t col, const float (&sum)[8]) {
    TO *row = (TO *)a.out + id * a.out_stride;
    Raw<TO> old;
    if (a.accumulate) {
        load8<SHORT>(old, row, col, a.dim);
        settle8<SHORT>(old, col, a.dim);
    } else old.clear();
    float v[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = sum[e] * a.scale + old.get(e);
    store8(row, col, a.dim, v);
}

/* L lanes to a step of the list and a tile of L*8 columns.  The places of the step and of what its last piece reaches beyond it
 * come in one trip to memory, then the rows, a set of them on its way while another is added up. */
template <typename TG, typename TO, int L, bool ACC, bool SHORT, bool ONCE> __global__ __launch_bounds__(kThreads) void embedding_sum_kernel(const GradArgs a) {
    static_assert(kListMost <= kWave, "a lane to a place");
    __shared__ Place list[L == kWave ? 1 : kThreads / L][kListMost];
    const uint32_t piece = 1u << a.log_piece, step = piece / 2;
    uint32_t team = threadIdx.x / L;
    if (L == kWave) team = (uint32_t)__builtin_amdgcn_readfirstlane((int)team);
    const uint32_t group = blockIdx.x * (kThreads / L) + team, lane = threadIdx.x % L, turn = group / a.tiles;
    const uint32_t col = (group - turn * a.tiles) * (L * 8) + lane * 8, begin = turn * step;
    Place held = {0, 0, 0, 0}; // of a whole wave each lane keeps a place
    if (L == kWave) {
        if (lane < step + piece && begin + lane < a.tokens) held = a.sorted[begin + lane];
    } else
        for (uint32_t i = lane; i < step + piece; i += L)
            if (begin + i < a.tokens) list[team][i] = a.sorted[begin + i];
    const uint32_t used = *a.used;
    __syncthreads();
    if (begin >= used) return;
    // pieces that begin here: from the first one's beginning to the last one's end, counted from `begin`
    const uint32_t here = used - begin < step ? used - begin : step;
    auto place = [&](uint32_t i) {
        if (L != kWave) return list[team][i];
        auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)i); };
        return Place{of(held.token), of(held.id), of(held.at), of(held.run)};
    };
    auto in = [&](const Place &p) { return p.at & (piece - 1); };
    auto rest = [&](const Place &p) { // from p to its piece's end
        const uint32_t left = p.run - p.at;
        return piece - in(p) < left ? piece - in(p) : left;
    };
    const Place head = place(0);
    const uint32_t first = in(head) ? rest(head) : 0;
    if (first >= here) return;
    const uint32_t end = here - 1 + rest(place(here - 1));
    auto ends = [&](const Place &p) { return in(p) == piece - 1 || p.at + 1 == p.run; };
    // Rows on their way: as many as the registers of two such sets hold.  No load of a set hangs on a condition (the last row stands
    // in for those past the end): with a known number under way, a wait for the first of them leaves the others alone.
    constexpr uint32_t kAhead = sizeof(TG) + (ACC ? sizeof(TO) : 0) <= 4 ? 4 : 2;
    struct Ahead {
        Raw<TG> grad[kAhead];
        Raw<TO> old[ACC ? kAhead : 1];
    };
    auto fetch = [&](Ahead &f, uint32_t at) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const Place p = place(at + k < end ? at + k : end - 1);
            load8<SHORT, ONCE>(f.grad[k], (const TG *)a.grad + p.token * a.grad_stride, col, a.dim);
            if (ACC) load8<SHORT>(f.old[k], (const TO *)a.out + p.id * a.out_stride, col, a.dim);
        }
    };
    // Sums are shifted into place at their end where a row ends inside the vector: adding up commutes with it.
    Raw<float> v;
    v.clear();
    auto add = [&](Ahead &f, uint32_t at) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            if (at + k >= end) break;
            const Place p = place(at + k);
            float sum[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                sum[e] = v.get(e) + f.grad[k].get(e);
                v.set(e, sum[e]);
            }
            if (!ends(p)) continue;
            const bool whole = p.run <= piece;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v.set(e, whole ? sum[e] * a.scale + (ACC ? f.old[k].get(e) : 0.0f) : sum[e]);
            settle8<SHORT>(v, col, a.dim);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) sum[e] = v.get(e);
            if (whole) store8((TO *)a.out + p.id * a.out_stride, col, a.dim, sum);
            else store8(a.partial + slot_of(begin + at + k - in(p), p.at < piece, a.log_piece) * a.padded, col, a.padded, sum);
            v.clear();
        }
    };
    Ahead one, two;
    fetch(one, first);
    for (uint32_t at = first; at < end; at += 2 * kAhead) {
        fetch(two, at + kAhead);
        add(one, at);
        fetch(one, at + 2 * kAhead);
        add(two, at + kAhead);
    }
}

/* Runs of several pieces: a wave looks for the one that begins in its places, as many as a piece is long, and sums its pieces
 * for 512 columns.  The pieces of a long one are shared out among the waves of the workgroup. */
constexpr uint32_t kTeam = 16;
template <typename TO, bool SHORT> __global__ __launch_bounds__(kTeam * kWave) void embedding_join_kernel(const GradArgs a, uint32_t first_team) {
    static_assert(kLogPieceMost <= 6, "a lane to a place");
    __shared__ Place runs[kTeam]; // token: where it begins
    __shared__ float sums[kTeam][512];
    const uint32_t used = *a.used, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, tile = blockIdx.x % a.tiles;
    const uint32_t begin = ((first_team + blockIdx.x / a.tiles) * kTeam + wave) << a.log_piece, piece = 1u << a.log_piece, col = tile * 512 + lane * 8;
    Place p = {0, 0, 1, 0};
    if (lane < piece && begin + lane < used) p = a.sorted[begin + lane];
    const bool found = p.at == 0 && p.run > piece; // one lane at most
    if (__ballot(found) == 0) p.run = 0;
    if (found || (p.run == 0 && lane == 0)) runs[wave] = Place{begin + lane, p.id, 0, p.run};
    __syncthreads();
    auto sum = [&](float (&v)[8], const Place &r, uint32_t from, uint32_t to) { // pieces of a run
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = 0.0f;
#pragma unroll 4
        for (uint32_t k = from; k < to; ++k) {
            Raw<float> s;
            load8<false>(s, (const float *)a.partial + slot_of(r.token + (k << a.log_piece), k == 0, a.log_piece) * a.padded, col, a.padded);
            settle8<false>(s, col, a.padded);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] += s.get(e);
        }
    };
    constexpr uint32_t kAlone = 8; // pieces that a wave sums by itself: they are all on their way at once
    float v[8];
    const Place own = runs[wave];
    const uint32_t pieces = (own.run + piece - 1) >> a.log_piece;
    if (own.run && pieces <= kAlone) {
        sum(v, own, 0, pieces);
        finish8<SHORT, TO>(a, own.id, col, v);
    }
    // the same for all waves: longer than that
    for (uint64_t left = __ballot(lane < kTeam && runs[lane < kTeam ? lane : 0].run > kAlone << a.log_piece); left; left &= left - 1) {
        const Place r = runs[__builtin_ctzll(left)];
        const uint32_t n = (r.run + piece - 1) >> a.log_piece, share = (n + kTeam - 1) / kTeam;
        sum(v, r, share * wave < n ? share * wave : n, share * (wave + 1) < n ? share * (wave + 1) : n);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) sums[wave][e * kWave + lane] = v[e];
        __syncthreads();
        if (wave == 0) {
#pragma unroll 3
            for (uint32_t o = 1; o < kTeam; ++o)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] += sums[o][e * kWave + lane];
            finish8<SHORT, TO>(a, r.id, col, v);
        }
        __syncthreads();
    }
}

/* A wave's zeros for SIZE bytes of a row of so many, an even number. */
template <uint32_t SIZE> __device__ __forceinline__ void zeros(char *row, uint32_t tile, uint32_t lane, uint64_t bytes) {
#pragma unroll
    for (uint32_t part = 0; part < SIZE; part += kWave * 16) {
        const uint64_t at = (uint64_t)tile * SIZE + part + lane * 16;
        if (at + 16 <= bytes) *(u32x4_at2 *)(row + at) = u32x4{0, 0, 0, 0};
        else
            for (uint64_t b = at; b < bytes; b += 2) *(uint16_t *)(row + b) = 0;
    }
}

/*
 * Few tokens: one launch.  A workgroup has a bucket's rows and a tile of 512 columns; each finds its tokens among all of them by
 * itself, writes its rows without a token, and sums the others: a row with up to kAloneFew tokens by one wave, one with more by
 * all four, their parts joined in the waves' order.  616 tokens into 49408 x 768 fp32 26 us, the speed of writing 152 MB of
 * zeros; 16 tokens into 1000 x 768 4.7 us.
 */
constexpr uint32_t kFewTokens = 1024;
constexpr uint32_t kFewLocals = 64; // rows of a bucket
constexpr uint32_t kAloneFew = 16;
template <typename TG, typename TO, bool ACC, bool SHORT> __global__ __launch_bounds__(kThreads) void embedding_few_kernel(const GradArgs a) {
    constexpr uint32_t kTeam = kThreads / kWave, kEach = kFewTokens / kThreads, kAhead = sizeof(TG) == 2 ? 16 : 8;
    __shared__ uint32_t counts[kFewLocals], numbers[kEach * kTeam], list[kFewTokens]; // list: token << 16 | local, ascending
    __shared__ float sums[kTeam][512];
    const uint32_t bucket = blockIdx.x / a.tiles, tile = blockIdx.x - bucket * a.tiles, mask = (1u << a.shift) - 1;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)), lane = threadIdx.x % kWave, col = tile * 512 + lane * 8;
    int64_t ids[kEach];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        const uint32_t t = k * kThreads + threadIdx.x;
        ids[k] = k * kThreads < a.tokens ? a.ids[t < a.tokens ? t : a.tokens - 1] : -1;
    }
    if (threadIdx.x < kFewLocals) counts[threadIdx.x] = 0;
    __syncthreads();
    uint64_t owns[kEach];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        const bool own = k * kThreads + threadIdx.x < a.tokens && a.counts(ids[k]) && ((uint32_t)ids[k] & mask) == bucket;
        if (own) atomicAdd(&counts[(uint32_t)ids[k] >> a.shift], 1u);
        owns[k] = __ballot(own);
        if (lane == 0) numbers[k * kTeam + wave] = (uint32_t)__popcll(owns[k]);
    }
    __syncthreads();
    uint32_t m = 0;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k)
#pragma unroll
        for (uint32_t w = 0; w < kTeam; ++w) {
            if (w == wave && (owns[k] >> lane & 1))
                list[m + (uint32_t)__popcll(owns[k] & ((1ull << lane) - 1))] = (k * kThreads + threadIdx.x) << 16 | (uint32_t)ids[k] >> a.shift;
            m += numbers[k * kTeam + w];
        }
    const uint32_t length = lane < kFewLocals ? counts[lane] : 0; // of the row with the lane's number
    const uint64_t exist = __ballot((lane << a.shift | bucket) < a.vocab && lane < a.locals);
    __syncthreads();
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (!ACC)
        for (uint64_t left = exist & ~__ballot(length != 0); left; left &= left - 1) {
            const uint32_t local = (uint32_t)__builtin_ctzll(left);
            if (local % kTeam == wave) zeros<512 * sizeof(TO)>((char *)a.out + (uint64_t)(local << a.shift | bucket) * a.out_stride * sizeof(TO), tile, lane, (uint64_t)a.dim * sizeof(TO));
        }
    // the tokens of a row, from the parts `from`, from + every and so on of the list, each of so many entries
    auto sum = [&](uint32_t local, uint32_t from, uint32_t every, uint32_t part) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = 0.0f;
        uint32_t n = 0, held = 0; // lane n of held: the n-th token that is under way
        auto flush = [&]() {
            Raw<TG> g[kAhead];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k)
                load8<SHORT>(g[k], (const TG *)a.grad + (uint32_t)__builtin_amdgcn_readlane((int)held, (int)(k < n ? k : n - 1)) * a.grad_stride, col, a.dim);
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) {
                if (k >= n) break;
                settle8<SHORT>(g[k], col, a.dim);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] += g[k].get(e);
            }
            n = 0;
        };
        for (uint32_t at = from * part; at < m; at += every * part) {
            const uint32_t entry = lane < part && at + lane < m ? list[at + lane] : 0xffffu;
            for (uint64_t left = __ballot((entry & 0xffffu) == local); left; left &= left - 1) {
                const uint32_t token = (uint32_t)__builtin_amdgcn_readlane((int)(entry >> 16), __builtin_ctzll(left));
                held = lane == n ? token : held;
                if (++n == kAhead) flush();
            }
        }
        if (n) flush();
    };
    uint32_t turn = 0;
    for (uint64_t left = __ballot(length != 0 && length <= kAloneFew); left; left &= left - 1, ++turn) {
        if (turn % kTeam != wave) continue;
        const uint32_t local = (uint32_t)__builtin_ctzll(left);
        sum(local, 0, 1, kWave);
        finish8<SHORT, TO>(a, local << a.shift | bucket, col, v);
    }
    for (uint64_t left = __ballot(length > kAloneFew); left; left &= left - 1) { // the same for all waves
        const uint32_t local = (uint32_t)__builtin_ctzll(left);
        sum(local, wave, kTeam, 16);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) sums[wave][e * kWave + lane] = v[e];
        __syncthreads();
        if (wave == 0) {
            for (uint32_t o = 1; o < kTeam; ++o)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] += sums[o][e * kWave + lane];
            finish8<SHORT, TO>(a, local << a.shift | bucket, col, v);
        }
        __syncthreads();
    }
}

uint32_t shift_of(uint64_t vocab, uint32_t most) { // for at most so many ids in a bucket
    uint32_t shift = 8;
    while (((vocab + (1ull << shift) - 1) >> shift) > most) ++shift;
    return shift;
}
/* One launch instead of three for few tokens, as long as the table is not so large that writing its zeros decides: whole rows from
 * fewer workgroups fill it faster then.  us, one launch | three, for 2, 300 and 1024 tokens:
 *   1000 x 768 bf16      5.2 | 8.9     6.4 | 13.6   10.9 | 14.8
 *   32000 x 2048 bf16    23.6 | 24.1   24.1 | 28.6  24.6 | 30.6
 *   49408 x 768 fp32     25.3 | 26.3   25.7 | 31.4  26.1 | 32.9
 *   44679 x 3630 fp32    182 | 142     182 | 148    183 | 150 */
bool is_few(uint64_t tokens, uint64_t vocab, uint64_t dim) {
    return tokens <= kFewTokens && vocab * dim <= 1u << 26 && ((dim + 511) / 512 << shift_of(vocab, kFewLocals)) <= 1u << 20;
}
uint64_t padded_of(uint64_t dim) { return (dim + 7) / 8 * 8; }

uint32_t lanes_of(uint64_t dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : 64; } // to a row in the sums

/* Short pieces where that is what it takes to have waves enough: 616 tokens of 768 took 7.9 us with pieces of 32, 4.7 with 8;
 * 32768 of 4096 84 with 32, 93 with 16, 124 with 8. */
constexpr uint32_t kLogPieceLeast = 3;
constexpr uint64_t kThreadsEnough = 2048 * kWave;
uint64_t threads_of(uint64_t dim) { // to a row in the sums, all tiles together
    const uint64_t lanes = lanes_of(dim);
    return (dim + lanes * 8 - 1) / (lanes * 8) * lanes;
}
uint32_t log_piece_of(uint64_t tokens, uint64_t dim) {
    uint32_t log_piece = kLogPieceMost;
    while (log_piece > kLogPieceLeast && (tokens >> (log_piece - 1)) * threads_of(dim) < kThreadsEnough) --log_piece;
    return log_piece;
}

/* The workspace: the number of places, the places, the sums of pieces; 16 bytes and multiples of them. */
constexpr uint64_t kHead = 16;
uint64_t partial_at(uint64_t tokens) { return kHead + tokens * sizeof(Place); }
/* For any number of tokens up to this one, so that a workspace that was made for the largest batch does for all.  Fewer tokens may be
 * cut into more pieces, shorter ones: at most as many as need the last threads that are wanted. */
uint64_t partial_bytes(uint64_t tokens, uint64_t dim) {
    const uint64_t own = tokens >> log_piece_of(tokens, dim), shortest = tokens >> kLogPieceLeast, wanted = (kThreadsEnough - 1) / threads_of(dim);
    const uint64_t fewer = shortest < wanted ? shortest : wanted, pieces = own > fewer ? own : fewer;
    return pieces ? 2 * (pieces + 1) * padded_of(dim) * sizeof(float) : 0;
}

template <typename TG, typename TO, int L, bool SHORT = false> void launch_sum(GradArgs a, hipStream_t s) {
    a.tiles = (a.dim + L * 8 - 1) / (L * 8);
    const uint32_t piece = 1u << a.log_piece, step = piece / 2;
    const uint64_t groups = (uint64_t)((a.tokens + step - 1) / step) * a.tiles;
    const dim3 grid((uint32_t)((groups + kThreads / L - 1) / (kThreads / L)));
    // Rows of grad are read once.  Where they and the table are more than the last cache holds, they go past it, so that they do not
    // push out the zeros that were just written: sums of 32768 x 4096 bf16 after 1 GB of zeros 117 -> 84 us.  Where they fit,
    // they may still be in it from the kernel that made them: 16384 x 1024 fp32 63 us past it, 57 through it.
    constexpr uint64_t kLastCache = 256u << 20;
    const bool once = L == kWave && (uint64_t)a.tokens * a.dim * sizeof(TG) + (uint64_t)a.vocab * a.dim * sizeof(TO) > kLastCache;
    void (*const kernel)(const GradArgs) =
        a.accumulate ? once ? embedding_sum_kernel<TG, TO, L, true, SHORT, L == kWave> : embedding_sum_kernel<TG, TO, L, true, SHORT, false>
                     : once ? embedding_sum_kernel<TG, TO, L, false, SHORT, L == kWave> : embedding_sum_kernel<TG, TO, L, false, SHORT, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a);
    if (a.tokens <= piece) return;
    a.tiles = (a.dim + 511) / 512;
    // teams of a launch, whose threads are counted in 32 bits; one launch up to 2^30 tokens of 512 columns
    const uint32_t teams = (a.tokens + kTeam * piece - 1) / (kTeam * piece), most = a.tiles < 1u << 21 ? (1u << 21) / a.tiles : 1;
    for (uint32_t at = 0; at < teams; at += most)
        hipLaunchKernelGGL((embedding_join_kernel<TO, SHORT>), dim3((teams - at < most ? teams - at : most) * a.tiles), dim3(kTeam * kWave), 0, s, a, at);
}
template <typename TG, typename TO> void launch_sums(const GradArgs &a, hipStream_t s) {
    const uint32_t lanes = lanes_of(a.dim);
    if (a.dim < 8) launch_sum<TG, TO, 8, true>(a, s);
    else if (lanes == 8) launch_sum<TG, TO, 8>(a, s);
    else if (lanes == 16) launch_sum<TG, TO, 16>(a, s);
    else if (lanes == 32) launch_sum<TG, TO, 32>(a, s);
    else launch_sum<TG, TO, 64>(a, s);
}

template <typename TG, typename TO> void launch_few(const GradArgs &a, uint32_t buckets, hipStream_t s) {
    void (*const kernel)(const GradArgs) =
        a.dim < 8 ? a.accumulate ? embedding_few_kernel<TG, TO, true, true> : embedding_few_kernel<TG, TO, false, true>
                  : a.accumulate ? embedding_few_kernel<TG, TO, true, false> : embedding_few_kernel<TG, TO, false, false>;
    hipLaunchKernelGGL(kernel, dim3(buckets * a.tiles), dim3(kThreads), 0, s, a);
}

} // namespace

int launch_embedding(const EriEmbedding &e, uint32_t compute_units, void *stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32 = e.dtype_tag == ERI_DTYPE_F32;
    constexpr uint64_t kMost = 1u << 22; // tokens of a launch
    for (uint64_t at = 0; at < e.tokens; at += kMost) {
        const LookupArgs a = {{(const char *)e.ids + at * (e.ids_64 ? 8 : 4), (uint32_t)e.ids_64}, e.table, (char *)e.out + at * e.out_stride * (f32 ? 4 : 2),
                              (uint32_t)(e.tokens - at < kMost ? e.tokens - at : kMost), (uint32_t)e.vocab, (uint32_t)e.dim, e.table_stride, e.out_stride, e.scale};
        if (f32) launch_lookup_of<float>(a, compute_units, s);
        else launch_lookup_of<bf16>(a, compute_units, s);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

uint64_t embedding_grad_workspace(uint64_t tokens, uint64_t vocab, uint64_t dim) {
    return is_few(tokens, vocab, dim) ? 0 : partial_at(tokens) + partial_bytes(tokens, dim);
}

int launch_embedding_grad(const EriEmbeddingGrad &e, void *stream) {
    char *ws = static_cast<char *>(e.workspace);
    // accumulating, there are no zeros to write: one launch as long as its workgroups, most of them with nothing to do, start faster than
    // two more launches.  300 tokens, one | three: 128000 x 1024 (4096 workgroups) 9.4 | 12.9 us, 88138 x 1272 (6144) 12.6 | 13.6,
    // 128000 x 2048 (8192) 15.6 | 13.7
    const bool few = is_few(e.tokens, e.vocab, e.dim) ||
                     (e.accumulate && e.tokens <= kFewTokens && ((e.dim + 511) / 512 << shift_of(e.vocab, kFewLocals)) <= 4096);
    GradArgs a = {{e.ids, (uint32_t)e.ids_64}, e.grad, e.out, (Place *)(ws + kHead), (uint32_t *)ws, (float *)(ws + partial_at(e.tokens)),
                  (uint32_t)e.tokens, (uint32_t)e.vocab, (uint32_t)e.dim, shift_of(e.vocab, few ? kFewLocals : kLocalMost), 0, (uint32_t)padded_of(e.dim), 0,
                  log_piece_of(e.tokens, e.dim), e.grad_stride, e.out_stride, e.padding_id, e.scale, (uint32_t)(e.accumulate != 0),
                  e.out_dtype == ERI_DTYPE_F32 ? 4u : 2u, 1};
    const bool g32 = e.grad_dtype == ERI_DTYPE_F32, o32 = e.out_dtype == ERI_DTYPE_F32;
    const uint32_t buckets = 1u << a.shift, used_buckets = buckets < a.vocab ? buckets : a.vocab;
    a.locals = (a.vocab + buckets - 1) >> a.shift;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (few) {
        a.tiles = (a.dim + 511) / 512;
        if (g32) o32 ? launch_few<float, float>(a, used_buckets, s) : launch_few<float, bf16>(a, used_buckets, s);
        else o32 ? launch_few<bf16, float>(a, used_buckets, s) : launch_few<bf16, bf16>(a, used_buckets, s);
        return (int)hipGetLastError();
    }
    while (a.lanes < kWave && a.lanes * 16ull < (uint64_t)a.dim * a.out_bytes) a.lanes *= 2;
    hipLaunchKernelGGL(embedding_sort_kernel, dim3(used_buckets), dim3(1024), kWaves * a.locals * 4, s, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || a.tokens == 0) return (int)err;
    if (g32) o32 ? launch_sums<float, float>(a, s) : launch_sums<float, bf16>(a, s);
    else o32 ? launch_sums<bf16, float>(a, s) : launch_sums<bf16, bf16>(a, s);
    return (int)hipGetLastError();
}

} // namespace eri_layers
