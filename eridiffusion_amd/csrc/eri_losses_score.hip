/*
 * Scores of tokens of include/eri_losses.h: one pass over the row with a running softmax, and the row's largest logits.
 *
 * Alternatives.  Every thread remembers the largest logit that it has seen and the vector that held it.  The k-th largest of these (value,
 * vector) pairs is a bound: k threads have an element above it or on it, so that whatever is below is not among the k largest, and only those k threads
 * can have seen one of them.  Each thread also leaves the largest of every few of its vectors in LDS (16 bits, rounded up); where that reaches the
 * bound, in little more than k places, the vectors are read once more, from the caches, and what passes the bound (about k elements) is sorted: 64 keys
 * of 64 bits to a wave, by a bitonic network over its lanes.
 */
#include "eri_losses_device.h"

namespace eri_losses {
namespace {

struct ScoreArgs {
    const void *logits, *ids;
    float *logprob, *entropy, *stats, *top;
    int64_t *top_ids;
    Sums *parts;    // of each slice of each row, where rows are cut
    Key *part_keys; // top of each
    uint64_t stride;
    uint32_t first, rows; // rows first .. rows-1
    uint32_t vocab, slices, shift; // 1 << shift vectors to a mark
    uint32_t top_n, ids_64;
    float c, inv_t;
};

/* What is written of a row, by one wave. */
template <typename T, bool ENT, bool TOP> __device__ __forceinline__ void finish(const ScoreArgs &a, uint64_t row, const Sums &r, Key k, float x, bool named, uint32_t lane) {
    const bool none = r.s == 0.0f; // NaN is something
    const float log_s = logf(r.s);
    if (lane == 0) {
        if (a.logprob) a.logprob[row] = !named ? 0.0f : none ? -kInf : (x - r.m) * a.inv_t - log_s;
        if (ENT) a.entropy[row] = none ? 0.0f : log_s - r.t * a.inv_t / r.s;
        a.stats[row * 2] = none ? -kInf : r.m;
        a.stats[row * 2 + 1] = log_s;
    }
    if (TOP && lane < a.top_n) {
        const bool nan = r.s != r.s;
        a.top[row * a.top_n + lane] = nan ? r.s : none ? -kInf : (value_of(k) - r.m) * a.inv_t - log_s;
        a.top_ids[row * a.top_n + lane] = nan ? lane : place_of(k);
    }
}

/* The token's logit, asked for early. */
template <typename T> __device__ __forceinline__ bool token_of(const ScoreArgs &a, uint64_t row, float *x) {
    if (!a.logprob) return false;
    const int64_t id = id_at(a.ids, a.ids_64, row);
    if (id < 0 || id >= (int64_t)a.vocab) return false;
    *x = at((const T *)a.logits + row * a.stride + id);
    return true;
}

/* What the threads of a workgroup tell each other about their elements. */
template <int TPR> constexpr uint32_t kMarks = TPR > (int)kWave ? 8192 : 1024; // largest values of a few vectors each, over all threads; a wave has shorter rows
template <int TPR> struct TopSpace {
    union {
        Key lists[TPR];      // until the bound is known
        uint32_t found[TPR]; // columns, 64 to a wave
    };
    Key bound;
    uint32_t places_n;
};
template <int TPR> struct Marks {
    uint16_t values[kMarks<TPR>] __attribute__((aligned(16)));
    uint16_t places[kWave * (kMarks<TPR> / TPR)]; // those that reach the bound: only 64 threads have any
};

/* The upper 16 bits of a value, rounded up. */
__device__ __forceinline__ uint32_t mark_of(float v, bool exact) {
    const uint32_t u = as_bits(v);
    return exact || (int32_t)u < 0 ? u >> 16 : (u + 0xffffu) >> 16;
}

/* The largest element of a thread and its first vector that holds it. */
struct Best {
    float value;
    uint32_t place;
    template <int E> __device__ __forceinline__ float take(const float (&v)[E], uint32_t vec) {
        const float m = largest(v, -kInf);
        if (m > value) value = m, place = vec;
        return m;
    }
};

/* A thread's first vector that holds anything of the row, which may begin some vectors after the first. */
template <int TPR, typename T> __device__ __forceinline__ uint32_t first_of(const Row<T> &row, uint32_t first, uint32_t t) {
    return first + t + (first + t < row.skip / kEach<T> ? TPR : 0);
}

/* The 64 largest of the lists that the waves have, in the first one. */
template <int TPR> __device__ __forceinline__ void join_lists(Key &k, Key *lists) {
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    if (TPR > (int)kWave) lists[t] = k;
#pragma unroll
    for (uint32_t half = TPR / kWave / 2; half > 0; half /= 2) {
        __syncthreads();
        if (wave < half) {
            merge64(k, lists[(wave + half) * kWave + (kWave - 1 - lane)], lane);
            if (half > 1) lists[t] = k;
        }
    }
}

/* The top_n-th largest of the threads' keys, 0 where fewer threads have one. */
template <int TPR> __device__ __forceinline__ Key bound_of(Key k, uint32_t top_n, TopSpace<TPR> &sp) {
    sort64(k, threadIdx.x % kWave);
    join_lists<TPR>(k, sp.lists);
    if (threadIdx.x == top_n - 1) sp.bound = k;
    if (threadIdx.x == 0) sp.places_n = 0;
    __syncthreads();
    return sp.bound;
}

/* For n things of each lane, n below 64, how many those before it have, and all lanes together. */
__device__ __forceinline__ uint32_t before_of(uint32_t n, uint32_t *total) {
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t b = 0; b < 6; ++b) {
        const uint64_t with = __ballot(n >> b & 1);
        before += __builtin_amdgcn_mbcnt_hi((uint32_t)(with >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)with, 0)) << b;
        all += (uint32_t)__popcll(with) << b;
    }
    *total = all;
    return before;
}
__device__ __forceinline__ void wave_sees() { // what its lanes have left in LDS
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* A wave's largest elements: columns are put down as they pass the bound, and sorted where 64 have come together. */
template <typename T> struct Largest {
    const Row<T> &row;
    const Key bound;
    uint32_t *const found; // 64 columns of this wave's
    const uint32_t lane;
    uint32_t n = 0;
    bool any = false;
    Key top = 0;
    __device__ __forceinline__ Largest(const Row<T> &r, Key b, uint32_t *all) : row(r), bound(b), found(all + threadIdx.x / kWave * kWave), lane(threadIdx.x % kWave) {}
    __device__ __forceinline__ void sort() {
        if (n == 0) return;
        wave_sees();
        Key k = 0;
        if (lane < n) {
            const uint32_t col = found[lane];
            k = key_of(at(row.from + row.skip + col), col);
        }
        wave_sees();
        sort64(k, lane);
        if (any) merge64(top, key_from(k, kWave - 1 - lane), lane);
        else top = k;
        any = true;
        n = 0;
    }
    /* The elements on or above the bound of N vectors, vec(i) with values v[i], of lanes that are active; all lanes of the wave call. */
    template <int N, int E, typename Vec> __device__ __forceinline__ void take(const float (&v)[N][E], bool active, Vec vec) {
        uint32_t which = 0;
        if (active) {
            const float least = bound ? value_of(bound) : -kInf;
            const uint32_t u = as_bits(least), next = (int32_t)u >= 0 ? u + 1 : u == 0x80000000u ? 1 : u - 1; // the next larger value
#pragma unroll
            for (uint32_t i = 0; i < (uint32_t)N; ++i) {
                const float from = bound == 0 || vec(i) <= place_of(bound) ? least : as_float(next); // later vectors lose a tie
                uint32_t these = 0;
#pragma unroll
                for (uint32_t e = 0; e < (uint32_t)E; ++e) these |= v[i][e] >= from ? 1u << e : 0u;
                if (!(vec(i) >= row.whole_from() && vec(i) < row.whole_to()))
#pragma unroll
                    for (uint32_t e = 0; e < (uint32_t)E; ++e)
                        if (!row.has(vec(i), e)) these &= ~(1u << e);
                which |= these << (i * E);
            }
        }
        uint32_t total, mine = (uint32_t)__popc(which), to = before_of(mine, &total);
        if (total == 0) return;
        if (n + total <= kWave) {
            for (to += n; which != 0; which &= which - 1) {
                const uint32_t b = (uint32_t)__builtin_ctz(which);
                found[to++] = row.col(vec(b / E), b % E);
            }
            n += total;
            return;
        }
        for (uint32_t b = 0; b < (uint32_t)(N * E); ++b) {
            const bool pass = which >> b & 1;
            const uint64_t with = __ballot(pass);
            const uint32_t more = (uint32_t)__popcll(with);
            if (n + more > kWave) sort();
            if (pass) found[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(with >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)with, 0))] = row.col(vec(b / E), b % E);
            n += more;
        }
    }
};

template <typename T, int TPR, bool ENT, bool TOP, bool ONCE> __global__ __launch_bounds__(TPR) void score_kernel(const ScoreArgs a) {
    constexpr int WAVES = TPR / (int)kWave;
    __shared__ Sums slots[WAVES];
    __shared__ char top_space[TOP ? sizeof(TopSpace<TPR>) : 1] __attribute__((aligned(16))), mark_space[TOP ? sizeof(Marks<TPR>) : 1] __attribute__((aligned(16)));
    TopSpace<TPR> &sp = *reinterpret_cast<TopSpace<TPR> *>(top_space);
    Marks<TPR> &marks = *reinterpret_cast<Marks<TPR> *>(mark_space);
    const uint32_t t = threadIdx.x, shift = a.shift;
    const uint64_t index = a.first + blockIdx.x;
    const Row<T> row((const T *)a.logits + index * a.stride, a.vocab);
    float x = 0.0f;
    const bool named = token_of<T>(a, index, &x);
    const uint32_t end = row.vectors();

    Sums r = {kLowest, 0.0f, 0.0f};
    Best best = {-kInf, first_of<TPR>(row, 0, t)};
    float run = -kInf;
    walk<TPR, ONCE>(row, 0, end, t, [&](auto &v, uint32_t at, bool) {
        constexpr uint32_t C = sizeof v / sizeof v[0];
        if (TOP)
#pragma unroll
            for (uint32_t k = 0; k < C; ++k) {
                run = fmaxf(run, best.take(v[k], at + k * TPR + t));
                if (k % 2 == 1 || k == C - 1) {
                    const uint32_t turn = at / TPR + k / 2 * 2;
                    marks.values[(turn >> shift) * TPR + t] = (uint16_t)mark_of(run, sizeof(T) == 2);
                    if (((turn + 2) & ((1u << shift) - 1)) == 0) run = -kInf;
                }
            }
        add<ENT>(r, v, a.c);
    });
    group_join<ENT, WAVES>(r, a.c, slots);
    Key k = 0;
    if (TOP) {
        const Key own = best.place < end ? key_of(best.value, best.place) : 0, bound = bound_of<TPR>(own, a.top_n, sp);
        const uint32_t turns = (end + TPR - 1) / TPR;
        const float least = bound ? value_of(bound) : -kInf;
        // one of top_n threads; marks of vectors behind the end hold anything, and lead nowhere
        for (uint32_t from = 0; from << shift < turns; from += 32) {
            uint32_t which = 0, total;
            if (own >= bound && own != 0)
                for (uint32_t i = 0; i < 32 && (from + i) << shift < turns; ++i)
                    if (as_float((uint32_t)marks.values[(from + i) * TPR + t] << 16) >= least) which |= 1u << i;
            uint32_t to = before_of((uint32_t)__popc(which), &total), base = 0;
            if (total == 0) continue;
            if (t % kWave == 0) base = atomicAdd(&sp.places_n, total);
            to += (uint32_t)__builtin_amdgcn_readfirstlane((int)base);
            for (; which != 0; which &= which - 1) marks.places[to++] = (uint16_t)((from + __builtin_ctz(which)) * TPR + t);
        }
        __syncthreads();
        Largest<T> found(row, bound, sp.found);
        const uint32_t total = sp.places_n << shift;
        for (uint32_t from = 0; from < total; from += TPR) {
            const uint32_t j = from + t, place = j < total ? marks.places[j >> shift] : 0, vec = place % TPR + ((place / TPR << shift) + (j & ((1u << shift) - 1))) * TPR;
            float v[1][kEach<T>];
            const bool real = j < total && vec < end;
            if (real) values_of(v[0], load_any<false>(row, vec));
            found.take(v, real, [&](uint32_t) { return vec; });
        }
        found.sort();
        k = found.top;
        join_lists<TPR>(k, reinterpret_cast<Key *>(marks.values)); // which are done with
    }
    if (t < kWave) finish<T, ENT, TOP>(a, index, r, k, x, named, t);
}

constexpr uint32_t kSliceThreads = 256;
template <typename T> constexpr uint32_t kSliceBatch = 32 / kEach<T>; // 32 columns to a thread

/* A slice of a row that a workgroup's registers hold: nothing is read twice. */
template <typename T, int TPR, bool ENT, bool TOP> __global__ __launch_bounds__(TPR) void score_slice_kernel(const ScoreArgs a) {
    constexpr int WAVES = TPR / (int)kWave;
    __shared__ Sums slots[WAVES];
    __shared__ char top_space[TOP ? sizeof(TopSpace<TPR>) : 1] __attribute__((aligned(16)));
    TopSpace<TPR> &sp = *reinterpret_cast<TopSpace<TPR> *>(top_space);
    const uint32_t t = threadIdx.x;
    const uint64_t index = a.first + blockIdx.x / a.slices;
    const Row<T> row((const T *)a.logits + index * a.stride, a.vocab);
    const uint32_t all = row.vectors(), first = blockIdx.x % a.slices * (kSliceBatch<T> * TPR);
    u32x4 raw[kSliceBatch<T>];
#pragma unroll
    for (uint32_t k = 0; k < kSliceBatch<T>; ++k) raw[k] = load_any<false>(row, first + k * TPR + t); // nothing where the row has no such vector
    float v[kSliceBatch<T>][kEach<T>];
#pragma unroll
    for (uint32_t k = 0; k < kSliceBatch<T>; ++k) values_of(v[k], raw[k]);
    Sums r = {kLowest, 0.0f, 0.0f};
    add<ENT>(r, v, a.c);
    group_join<ENT, WAVES>(r, a.c, slots);
    Key k = 0;
    if (TOP) {
        Best best = {-kInf, first_of<TPR>(row, first, t)};
#pragma unroll
        for (uint32_t i = 0; i < kSliceBatch<T>; ++i) best.take(v[i], first + i * TPR + t);
        const Key own = best.place < all ? key_of(best.value, best.place) : 0;
        Key bound = own;
        if (a.top_n <= kWave / 2) { // each wave by itself: it keeps about as many elements as are wanted, and the waves need not wait for each other
            sort64(bound, t % kWave);
            bound = (Key)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bound >> 32), (int)a.top_n - 1) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bound, (int)a.top_n - 1);
        } else bound = bound_of<TPR>(own, a.top_n, sp);
        Largest<T> found(row, bound, sp.found);
        found.take(v, own >= bound && own != 0, [&](uint32_t i) { return first + i * TPR + t; });
        found.sort();
        k = found.top;
        __shared__ Key lists[TPR];
        join_lists<TPR>(k, lists);
    }
    if (t == 0) a.parts[blockIdx.x] = r;
    if (TOP && t < a.top_n) a.part_keys[(uint64_t)blockIdx.x * a.top_n + t] = k;
}

/* Joins the slices of a row: 8 waves, each with an eighth of the lists. */
template <typename T, bool ENT, bool TOP> __global__ __launch_bounds__(512) void score_join_kernel(const ScoreArgs a) {
    __shared__ Key lists[512];
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const uint64_t index = a.first + blockIdx.x;
    const uint32_t from = blockIdx.x * a.slices;
    float x = 0.0f;
    const bool named = token_of<T>(a, index, &x);
    Key k = 0;
    if (TOP) {
        Key list[kSlicesMost / 8];
#pragma unroll
        for (uint32_t i = 0; i < kSlicesMost / 8; ++i) {
            const uint32_t s = i * 8 + wave, place = i ? kWave - 1 - lane : lane; // the others upside down, for the merge
            list[i] = s < a.slices && place < a.top_n ? a.part_keys[(uint64_t)(from + s) * a.top_n + place] : 0;
        }
        k = list[0];
#pragma unroll
        for (uint32_t i = 1; i < kSlicesMost / 8; ++i)
            if (i * 8 < a.slices) merge64(k, list[i], lane);
        lists[t] = k;
#pragma unroll
        for (uint32_t half = 4; half > 0; half /= 2) {
            __syncthreads();
            if (wave < half) {
                merge64(k, lists[(wave + half) * kWave + (kWave - 1 - lane)], lane);
                lists[t] = k;
            }
        }
    }
    if (wave != 0) return;
    Sums r = {kLowest, 0.0f, 0.0f};
    if (lane < a.slices) r = a.parts[from + lane];
    wave_join<ENT>(r, a.c);
    finish<T, ENT, TOP>(a, index, r, k, x, named, lane);
}

uint32_t slices_of(uint64_t vocab) { return (uint32_t)((vocab + 63 + 32 * kSliceThreads - 1) / (32 * kSliceThreads)); } // up to 63 columns of the first are none
uint64_t parts_most(uint64_t rows, uint64_t vocab) {
    const uint64_t slices = slices_of(vocab);
    return vectors_most<float>(vocab) > kLong ? (rows < kFew ? rows : kFew) * (slices < kSlicesMost ? slices : kSlicesMost) : 0;
}

/* Threads to a row.  us for a call, bf16 and f32, with and without 20 alternatives:
 *                        256 threads              1024                     slices, joined
 *     1 row  of  4000 vectors    6.0  8.7            6.2  9.8                 7.7  9.3
 *     1          8000            6.1  9.7            5.9  9.4                 7.7  8.9
 *     1         16000           10.3 16.7            8.7 15.0                 7.9  9.3
 *    64         16000           12.8 19.2            9.8 16.2                 7.7 13.3
 *   128         16000           14.4 21.0           10.5 16.8                 9.9 18.7
 *   256         32000           26.7 34.4           21.6 27.6                24.4 41.6
 *   400         16000           18.4 25.3           20.2 33.1                19.8 39.5
 * and a wave to a row, bf16:
 * 16384 rows of  375 vectors   23.6 75.6, not 18.2 30.9;   750   35.7 88.9, 37.0 46.5;   1500   60.2 113,  71.7 84.5
 *   200          375            6.1  7.0       6.1  7.2;   1500    5.8  7.6,  5.9  9.3
 * With 64 alternatives each lane of a wave is above the bound: 16384 rows of 750 vectors 93.3, not 96.5, of 1500 129 and 172; with 48 and fewer a wave wins. */
template <typename T, bool ENT, bool TOP> void launch(ScoreArgs &a, uint64_t all_rows, hipStream_t s) {
    const uint32_t rows = a.rows - a.first, n = vectors_most<T>(a.vocab);
    const bool large = all_rows * a.vocab * sizeof(T) > kCache; // for a wave with alternatives it does not pay: their vectors are read again (65536 x 4000 132 us, so 147)
#define ERI_SCORE(TPR, ONCE) \
    do { \
        for (a.shift = 1; n / TPR >> a.shift >= kMarks<TPR> / TPR;) ++a.shift; \
        hipLaunchKernelGGL((score_kernel<T, TPR, ENT, TOP, ONCE>), dim3(rows), dim3(TPR), 0, s, a); \
    } while (0)
    a.slices = slices_of(a.vocab);
    if (n > kLong && all_rows <= kFew && a.slices <= kSlicesMost) {
        hipLaunchKernelGGL((score_slice_kernel<T, kSliceThreads, ENT, TOP>), dim3(rows * a.slices), dim3(kSliceThreads), 0, s, a);
        hipLaunchKernelGGL((score_join_kernel<T, ENT, TOP>), dim3(rows), dim3(TOP ? 512 : 64), 0, s, a);
    } else if (n <= 256 || (all_rows >= 1024 && n <= (TOP && a.top_n <= 48 ? 2048u : 512u))) {
        if constexpr (TOP) ERI_SCORE(64, false);
        else if (large) ERI_SCORE(64, true);
        else ERI_SCORE(64, false);
    } else if (n > kLong && all_rows <= 256) ERI_SCORE(1024, false);
    else if (large) ERI_SCORE(256, true);
    else ERI_SCORE(256, false);
#undef ERI_SCORE
}
template <typename T> void launch_of(ScoreArgs &a, uint64_t rows, hipStream_t s) {
    if (a.entropy) a.top_n ? launch<T, true, true>(a, rows, s) : launch<T, true, false>(a, rows, s);
    else a.top_n ? launch<T, false, true>(a, rows, s) : launch<T, false, false>(a, rows, s);
}

} // namespace

uint64_t token_logprobs_workspace(uint64_t rows, uint64_t vocab, uint32_t top) { return parts_most(rows, vocab) * (16 + (uint64_t)top * sizeof(Key)); }

int launch_token_logprobs(const EriTokenLogprobs &e, void *stream) {
    ScoreArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.logprob = e.ids ? e.logprob : nullptr, a.entropy = e.entropy, a.stats = e.stats, a.top = e.top, a.top_ids = e.top_ids;
    a.stride = e.logits_stride, a.vocab = (uint32_t)e.vocab, a.top_n = (uint32_t)e.top_n, a.ids_64 = (uint32_t)e.ids_64;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
    a.parts = (Sums *)e.workspace; // 16 bytes to each, then the keys
    a.part_keys = (Key *)((char *)e.workspace + parts_most(e.rows, e.vocab) * 16);
    constexpr uint32_t kMost = 1u << 21; // rows of a launch
    for (uint64_t first = 0; first < e.rows; first += kMost) {
        a.first = (uint32_t)first;
        a.rows = (uint32_t)(e.rows - first < kMost ? e.rows : first + kMost);
        if (e.dtype_tag == ERI_DTYPE_F32) launch_of<float>(a, e.rows, static_cast<hipStream_t>(stream));
        else launch_of<bf16>(a, e.rows, static_cast<hipStream_t>(stream));
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

} // namespace eri_losses
