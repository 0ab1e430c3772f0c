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

constexpr uint32_t kFound = 256; // elements that pass the bound and are kept at a time

struct ScoreArgs {
    const void *logits, *ids;
    float *logprob, *entropy, *stats, *top;
    int64_t *top_ids;
    Sums *parts;    // of each slice of each row, where rows are cut
    Key *part_keys; // top of each
    uint64_t stride;
    uint32_t first, rows; // rows first .. rows-1
    uint32_t vocab, slices, per; // per: vectors to a slice
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

constexpr uint32_t kMarks = 8192; // largest values of a few vectors each, over all threads
template <int TPR> struct TopSpace {
    uint16_t marks[kMarks];
    union {
        Key lists[TPR];
        Key found[kFound];
    };
    uint16_t places[kWave * (kMarks / TPR)]; // marks that reach the bound: only k threads have any
    Key bound;
    uint32_t places_n, count;
};

/* The upper 16 bits of a value, rounded up. */
__device__ __forceinline__ uint32_t mark_of(float v, bool exact) {
    const uint32_t u = as_bits(v);
    return exact || (int32_t)u < 0 ? u >> 16 : (u + 0xffffu) >> 16;
}

/* What a thread knows of its elements: the largest, its first vector that holds it, and the largest of every `each` of its vectors (a power
 * of two), which it leaves in marks[turn / each]. */
template <typename T, int TPR> struct Seen {
    float best, run;
    uint32_t place;
    __device__ __forceinline__ void take(const float (&v)[8], uint32_t vec) {
        const float m = largest(v);
        if (m > best) best = m, place = vec;
        run = fmaxf(run, m);
    }
    /* after each one or two vectors from `turn` on */
    __device__ __forceinline__ void mark(TopSpace<TPR> &sp, uint32_t turn, uint32_t shift) {
        sp.marks[(turn >> shift) * TPR + threadIdx.x] = (uint16_t)mark_of(run, sizeof(T) == 2);
        if (((turn + 2) & ((1u << shift) - 1)) < 2) run = -kInf;
    }
};

/* The row's (or slice's) largest elements in the lanes of the first wave, in descending order; vectors first .. end-1 are dealt to the threads in turn. */
template <typename T, int TPR> __device__ __forceinline__ Key largest_of(const T *row, const Seen<T, TPR> &seen, uint32_t shift, uint32_t first, uint32_t end, uint32_t vocab, uint32_t top_n, TopSpace<TPR> &sp) {
    constexpr uint32_t WAVES = TPR / kWave;
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = t / kWave, whole = vocab / 8;
    const Key own = first + t < end ? key_of(seen.best, seen.place) : 0;
    Key k = own;
    sort64(k, lane);
    if (WAVES > 1) sp.lists[t] = k;
    for (uint32_t half = WAVES / 2; half > 0; half /= 2) {
        __syncthreads();
        if (wave < half) {
            merge64(k, sp.lists[(wave + half) * kWave + (kWave - 1 - lane)], lane);
            sp.lists[t] = k;
        }
    }
    if (t == top_n - 1) sp.bound = k; // 0, which all pass, where fewer threads have seen anything
    if (t == 0) sp.places_n = 0;
    __syncthreads();
    const Key bound = sp.bound;
    const uint32_t turns = (end - first + TPR - 1) / TPR;
    const float least = bound ? value_of(bound) : -kInf;
    if (own >= bound && own != 0) // one of top_n threads; marks of vectors behind the end hold anything, and lead nowhere
        for (uint32_t i = 0; i << shift < turns; ++i)
            if (as_float((uint32_t)sp.marks[i * TPR + t] << 16) >= least) sp.places[atomicAdd(&sp.places_n, 1u)] = (uint16_t)(i * TPR + t);
    __syncthreads();
    const uint32_t total = sp.places_n << shift;
    uint32_t per = total;
    Key top = 0;
    for (uint32_t from = 0; from < total;) {
        if (t == 0) sp.count = 0;
        __syncthreads();
        const uint32_t to = per < total - from ? from + per : total;
        for (uint32_t j = from + t; j < to; j += TPR) {
            const uint32_t place = sp.places[j >> shift], vec = first + place % TPR + ((place / TPR << shift) + (j & ((1u << shift) - 1))) * TPR;
            if (vec >= end) continue;
            float v[8];
            if (vec < whole) {
                Raw<T> r;
                r.load(row + (uint64_t)vec * 8);
                values_of(v, r);
            } else load_last(v, row + (uint64_t)vec * 8, vocab % 8);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (vec * 8 + e < vocab && key_of(v[e], vec) >= bound) {
                    const uint32_t i = atomicAdd(&sp.count, 1u);
                    if (i < kFound) sp.found[i] = key_of(v[e], vec * 8 + e);
                }
        }
        __syncthreads();
        const uint32_t c = sp.count;
        __syncthreads();
        if (c > kFound) { // far more on one side of a tie than there are threads: again from the start, so few vectors at a time that they fit
            per = kFound / 8;
            continue;
        }
        if (t < kWave)
            for (uint32_t i = 0; i < c; i += kWave) {
                Key f = i + lane < c ? sp.found[i + lane] : 0;
                sort64(f, lane);
                if (i == 0 && from == 0) top = f;
                else merge64(top, key_from(f, kWave - 1 - lane), lane);
            }
        __syncthreads();
        from = to;
    }
    return top;
}

template <typename T, int TPR, bool ENT, bool TOP, bool SPLIT> __global__ __launch_bounds__(TPR) void score_kernel(const ScoreArgs a) {
    constexpr int WAVES = TPR / (int)kWave;
    __shared__ Sums slots[WAVES];
    __shared__ char space[TOP ? sizeof(TopSpace<TPR>) : 1] __attribute__((aligned(16)));
    const uint32_t t = threadIdx.x, slice = SPLIT ? blockIdx.x % a.slices : 0;
    const uint64_t index = a.first + (SPLIT ? blockIdx.x / a.slices : blockIdx.x);
    const T *row = (const T *)a.logits + index * a.stride;
    float x = 0.0f;
    const bool named = !SPLIT && token_of<T>(a, index, &x);
    const uint32_t whole = a.vocab / 8, all = (a.vocab + 7) / 8;
    const uint32_t first = SPLIT ? slice * a.per : 0, end = SPLIT && all - first > a.per ? first + a.per : all, last = end < whole ? end : whole;

    Sums r = {kLowest, 0.0f, 0.0f};
    Seen<T, TPR> seen = {-kInf, -kInf, first + t};
    TopSpace<TPR> &sp = *reinterpret_cast<TopSpace<TPR> *>(space);
    uint32_t shift = 1; // so that the marks suffice
    while (TOP && (a.per / TPR) >> shift >= kMarks / TPR) ++shift;
    walk<TPR>(row, first, last, t, [&](auto &v, uint32_t at, bool) {
        constexpr uint32_t C = sizeof v / sizeof v[0];
        if (TOP)
#pragma unroll
            for (uint32_t k = 0; k < C; ++k) {
                seen.take(v[k], at + k * TPR + t);
                if (k % 2 == 1 || k == C - 1) seen.mark(sp, (at - first) / TPR + k / 2 * 2, shift);
            }
        add<ENT>(r, v, a.c);
    });
    if (end > whole && t == (whole - first) % TPR) { // the row's last vector, of less than eight elements
        float v[1][8];
        load_last(v[0], row + (uint64_t)whole * 8, a.vocab % 8);
        if (TOP) {
            const uint32_t turn = (whole - first) / TPR;
            const float m = largest(v[0]);
            seen.take(v[0], whole);
            // its mark may hold vectors before it
            if (turn & ((1u << shift) - 1)) seen.run = fmaxf(m, as_float((uint32_t)sp.marks[(turn >> shift) * TPR + t] << 16));
            else seen.run = m;
            sp.marks[(turn >> shift) * TPR + t] = (uint16_t)mark_of(seen.run, sizeof(T) == 2);
        }
        add<ENT>(r, v, a.c);
    }
    group_join<ENT, WAVES>(r, a.c, slots);
    Key k = 0;
    if (TOP) k = largest_of<T, TPR>(row, seen, shift, first, end, a.vocab, a.top_n, sp);
    if (t >= kWave) return;
    if (SPLIT) {
        if (t == 0) a.parts[blockIdx.x] = r;
        if (TOP && t < a.top_n) a.part_keys[(uint64_t)blockIdx.x * a.top_n + t] = k;
    } else finish<T, ENT, TOP>(a, index, r, k, x, named, t);
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
        for (uint32_t s = wave; s < a.slices; s += 8) {
            const uint32_t up = kWave - 1 - lane;
            merge64(k, up < a.top_n ? a.part_keys[(uint64_t)(from + s) * a.top_n + up] : 0, lane);
        }
        lists[t] = k;
        __syncthreads();
        if (wave == 0)
            for (uint32_t w = 1; w < 8; ++w) merge64(k, lists[w * kWave + (kWave - 1 - lane)], lane);
    }
    if (wave != 0) return;
    Sums r = {kLowest, 0.0f, 0.0f};
    if (lane < a.slices) r = a.parts[from + lane];
    wave_join<ENT>(r, a.c);
    finish<T, ENT, TOP>(a, index, r, k, x, named, lane);
}

/* Slices of a row.  Rows that fill the chip by themselves are not cut. */
constexpr uint32_t kFill = 1024, kSlicesMost = 64;
uint32_t slices_most(uint64_t vocab) {
    const uint64_t n = (vocab + 7) / 8 / 512;
    return n < 1 ? 1 : n > kSlicesMost ? kSlicesMost : (uint32_t)n;
}
uint32_t slices_of(uint64_t rows, uint64_t vocab) {
    const uint64_t n = kFill / rows, most = slices_most(vocab);
    return n < 2 ? 1 : (uint32_t)(n < most ? n : most);
}

template <typename T, bool ENT, bool TOP> void launch(const ScoreArgs &a, hipStream_t s) {
    const uint32_t rows = a.rows - a.first;
    if (a.slices > 1) {
        hipLaunchKernelGGL((score_kernel<T, 256, ENT, TOP, true>), dim3(rows * a.slices), dim3(256), 0, s, a);
        hipLaunchKernelGGL((score_join_kernel<T, ENT, TOP>), dim3(rows), dim3(TOP ? 512 : 64), 0, s, a);
    } else if (a.vocab <= 2048) hipLaunchKernelGGL((score_kernel<T, 64, ENT, TOP, false>), dim3(rows), dim3(64), 0, s, a);
    else hipLaunchKernelGGL((score_kernel<T, 256, ENT, TOP, false>), dim3(rows), dim3(256), 0, s, a);
}
template <typename T> void launch_of(const ScoreArgs &a, hipStream_t s) {
    if (a.entropy) a.top_n ? launch<T, true, true>(a, s) : launch<T, true, false>(a, s);
    else a.top_n ? launch<T, false, true>(a, s) : launch<T, false, false>(a, s);
}

} // namespace

uint64_t token_logprobs_workspace(uint64_t rows, uint64_t vocab, uint32_t top) {
    const uint64_t most = slices_most(vocab), parts = rows * most < kFill ? rows * most : kFill;
    return most > 1 ? parts * (16 + (uint64_t)top * sizeof(Key)) : 0;
}

int launch_token_logprobs(const EriTokenLogprobs &e, void *stream) {
    ScoreArgs a = {};
    a.logits = e.logits, a.ids = e.ids, a.logprob = e.ids ? e.logprob : nullptr, a.entropy = e.entropy, a.stats = e.stats, a.top = e.top, a.top_ids = e.top_ids;
    a.stride = e.logits_stride, a.vocab = (uint32_t)e.vocab, a.top_n = (uint32_t)e.top_n, a.ids_64 = (uint32_t)e.ids_64;
    a.c = (float)(kLog2e / e.temperature), a.inv_t = (float)(1.0 / e.temperature);
    const uint32_t n = (a.vocab + 7) / 8, want = slices_of(e.rows, e.vocab);
    a.per = ((n + want - 1) / want + 255) / 256 * 256;
    a.slices = (n + a.per - 1) / a.per;
    a.part_keys = (Key *)e.workspace; // keys first: they need more alignment
    a.parts = (Sums *)(a.part_keys + (a.slices > 1 ? e.rows * a.slices * e.top_n : 0));
    constexpr uint32_t kMost = 1u << 21; // rows of a launch
    for (uint64_t first = 0; first < e.rows; first += kMost) {
        a.first = (uint32_t)first;
        a.rows = (uint32_t)(e.rows - first < kMost ? e.rows : first + kMost);
        if (e.dtype_tag == ERI_DTYPE_F32) launch_of<float>(a, static_cast<hipStream_t>(stream));
        else launch_of<bf16>(a, static_cast<hipStream_t>(stream));
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

} // namespace eri_losses
