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

/* L lanes to a row, U rows at a time in each thread's registers. */
template <typename T, int L, int U> __global__ __launch_bounds__(kThreads) void embedding_kernel(const LookupArgs a) {
    constexpr uint32_t kRows = kThreads / L;
    const uint32_t first = blockIdx.x * kRows * U + threadIdx.x / L, lane = threadIdx.x % L;
    const T *row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t t = first + u * kRows;
        const int64_t id = t < a.tokens ? a.ids[t] : -1;
        row[u] = (uint64_t)id < a.vocab ? (const T *)a.table + id * a.table_stride : nullptr;
    }
    for (uint32_t col = lane * 8; col < a.dim; col += L * 8) {
        Raw<T> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row[u]) load8(r[u], row[u], col, a.dim);
            else r[u].clear();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t t = first + u * kRows;
            float v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] = row[u] ? r[u].get(e) * a.scale : 0.0f;
            if (t < a.tokens) store8((T *)a.out + t * a.out_stride, col, a.dim, v);
        }
    }
}

template <typename T, int L> void launch_lookup(const LookupArgs &a, uint32_t compute_units, hipStream_t s) {
    constexpr uint32_t kRows = kThreads / L;
    if (a.tokens / (kRows * 4) >= compute_units * 4) // four rows a thread where that still fills the chip
        hipLaunchKernelGGL((embedding_kernel<T, L, 4>), dim3((a.tokens + kRows * 4 - 1) / (kRows * 4)), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((embedding_kernel<T, L, 1>), dim3((a.tokens + kRows - 1) / kRows), dim3(kThreads), 0, s, a);
}
template <typename T> void launch_lookup_of(const LookupArgs &a, uint32_t compute_units, hipStream_t s) {
    if (a.dim <= 64) launch_lookup<T, 8>(a, compute_units, s);
    else if (a.dim <= 256) launch_lookup<T, 32>(a, compute_units, s);
    else if (a.dim <= 1024) launch_lookup<T, 128>(a, compute_units, s);
    else launch_lookup<T, 256>(a, compute_units, s);
}

// ---------------------------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------------------------

/*
 * Ids are dealt to K = 2^shift buckets by their low bits, a workgroup to a bucket.  It reads all ids twice, in order:
 * the first time it counts its own ones, each wave for its share of the tokens; the second time it writes the tokens of
 * each of its ids, in ascending order, to its part of `order`.  Where that part begins, it has counted too, as the
 * number of tokens in the buckets before it: no workgroup waits for another.  Then it writes its rows of the gradient:
 * zeros where no token names the row, the sum of up to kFew rows of grad.  Rows with more tokens go to a second kernel,
 * which spreads each over many workgroups.
 */
constexpr uint32_t kWaves = 16;       // of a bucket's workgroup
constexpr uint32_t kLocalMost = 1024; // ids of a bucket
constexpr uint32_t kFew = 64;

struct Heavy { // a row with more than kFew tokens
    uint32_t id, start, count, unused;
};

struct GradArgs {
    Ids ids;
    const void *grad;
    void *out;
    uint32_t *order;  // tokens numbers
    Heavy *heavy;     // bucket b's from place heavy_first[b] on
    uint32_t *heavy_first, *heavy_count; // one per bucket
    uint32_t tokens, vocab, dim, shift, locals;
    uint64_t grad_stride, out_stride;
    int64_t padding_id;
    float scale;
    uint32_t accumulate;
    __device__ __forceinline__ bool counts(int64_t id) const { return (uint64_t)id < vocab && id != padding_id; }
};

template <typename TO> __device__ __forceinline__ void finish8(const GradArgs &a, uint32_t id, uint32_t col, float (&v)[8]) {
    TO *row = (TO *)a.out + id * a.out_stride;
    Raw<TO> old;
    if (a.accumulate) load8(old, row, col, a.dim);
    else old.clear();
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) v[e] = v[e] * a.scale + old.get(e);
    store8(row, col, a.dim, v);
}

template <typename TG, typename TO, int L> __global__ __launch_bounds__(1024) void embedding_grad_kernel(const GradArgs a) {
    extern __shared__ uint32_t counts[]; // kWaves x locals: first counts, then where the wave's next token of that id goes
    __shared__ uint32_t starts[kLocalMost], lengths[kLocalMost], part[kWaves], before[kWaves], n_heavy;
    const uint32_t bucket = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, mask = (1u << a.shift) - 1;
    if (bucket >= a.vocab) return;
    for (uint32_t i = threadIdx.x; i < kWaves * a.locals; i += 1024) counts[i] = 0;
    if (threadIdx.x == 0) n_heavy = 0;
    __syncthreads();

    // count
    const uint32_t share = (a.tokens + kWaves * kWave - 1) / (kWaves * kWave) * kWave;
    const uint32_t from = wave * share, to = from + share < a.tokens ? from + share : a.tokens;
    uint32_t *mine = counts + wave * a.locals, lower = 0;
#pragma unroll 4
    for (uint32_t t = from + lane; t < to; t += kWave) {
        const int64_t id = a.ids[t];
        if (!a.counts(id)) continue;
        const uint32_t b = (uint32_t)id & mask;
        if (b == bucket) atomicAdd(&mine[(uint32_t)id >> a.shift], 1u);
        lower += b < bucket;
    }
    for (int d = 1; d < 64; d *= 2) lower += __shfl_xor(lower, d);
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
    uint32_t start = base + upto - total;
    for (uint32_t w = 0; w < wave; ++w) start += part[w];
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

    // order: each wave for its share; of several tokens in one step, an id at a time
    for (uint32_t at = from; at < to; at += kWave) {
        const int64_t id = at + lane < to ? a.ids[at + lane] : -1;
        const bool own = a.counts(id) && ((uint32_t)id & mask) == bucket;
        uint64_t left = __ballot(own);
        while (left) {
            const uint32_t local = (uint32_t)__builtin_amdgcn_readlane((int)((uint32_t)id >> a.shift), __builtin_ctzll(left));
            const bool same = own && ((uint32_t)id >> a.shift) == local;
            const uint64_t all = __ballot(same);
            uint32_t place = 0;
            if (lane == 0) place = atomicAdd(&mine[local], (uint32_t)__popcll(all));
            place = (uint32_t)__builtin_amdgcn_readfirstlane((int)place);
            if (same) a.order[place + (uint32_t)__popcll(all & ((1ull << lane) - 1))] = at + lane;
            left &= ~all;
        }
    }
    __syncthreads();

    // rows: L lanes to each
    const uint32_t sub = lane % L;
    for (uint32_t local = threadIdx.x / L; local < a.locals; local += 1024 / L) {
        const uint32_t id = local << a.shift | bucket, n = lengths[local], begin = starts[local];
        if (id >= a.vocab || (n == 0 && a.accumulate)) continue;
        if (n > kFew) {
            if (sub == 0) a.heavy[base / (kFew + 1) + atomicAdd(&n_heavy, 1u)] = Heavy{id, begin, n, 0};
            continue;
        }
        for (uint32_t col = sub * 8; col < a.dim; col += L * 8) {
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
            for (uint32_t j = 0; j < n; ++j) {
                Raw<TG> g;
                load8(g, (const TG *)a.grad + a.order[begin + j] * a.grad_stride, col, a.dim);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] += g.get(e);
            }
            finish8<TO>(a, id, col, v);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        a.heavy_first[bucket] = base / (kFew + 1);
        a.heavy_count[bucket] = n_heavy;
    }
}

/* The rows with many tokens: 64 columns of one to a workgroup, eight lanes to a token's part of them. */
constexpr uint32_t kHeavyThreads = 512;
template <typename TG, typename TO> __global__ __launch_bounds__(kHeavyThreads) void embedding_grad_heavy_kernel(const GradArgs a, uint32_t buckets) {
    __shared__ float sums[kHeavyThreads / 8][64];
    const uint32_t group = threadIdx.x / 8, in = threadIdx.x % 8 * 8, col = blockIdx.x * 64 + in;
    for (uint32_t bucket = blockIdx.y; bucket < buckets; bucket += gridDim.y)
    for (uint32_t i = 0, n = a.heavy_count[bucket], first = a.heavy_first[bucket]; i < n; ++i) {
        const Heavy h = a.heavy[first + i];
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
        for (uint32_t j = group; j < h.count; j += kHeavyThreads / 8) {
            Raw<TG> g;
            load8(g, (const TG *)a.grad + a.order[h.start + j] * a.grad_stride, col, a.dim);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] += g.get(e);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) sums[group][in + e] = v[e];
        __syncthreads();
        if (threadIdx.x < 8) {
            for (uint32_t p = 1; p < kHeavyThreads / 8; ++p)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] += sums[p][in + e];
            finish8<TO>(a, h.id, col, v);
        }
    }
}

uint32_t shift_of(uint64_t vocab) {
    uint32_t shift = 8;
    while (((vocab + (1ull << shift) - 1) >> shift) > kLocalMost) ++shift;
    return shift;
}

/* The workspace: order, heavy, heavy_first, heavy_count, each at a multiple of 16 bytes. */
struct Workspace {
    uint64_t heavy, first, count, bytes;
    Workspace(uint64_t tokens, uint64_t vocab) {
        heavy = (tokens * 4 + 15) / 16 * 16;
        first = heavy + (tokens / (kFew + 1)) * sizeof(Heavy);
        count = first + (4ull << shift_of(vocab));
        bytes = count + (4ull << shift_of(vocab));
    }
};

template <typename TG, typename TO> void launch_grad(const GradArgs &a, hipStream_t s) {
    const uint32_t buckets = 1u << a.shift, lds = kWaves * a.locals * 4;
    const uint32_t grid = buckets < a.vocab ? buckets : a.vocab;
#define ERI_EMB_GRAD(L) hipLaunchKernelGGL((embedding_grad_kernel<TG, TO, L>), dim3(grid), dim3(1024), lds, s, a)
    if (a.dim <= 64) ERI_EMB_GRAD(8);
    else if (a.dim <= 128) ERI_EMB_GRAD(16);
    else if (a.dim <= 256) ERI_EMB_GRAD(32);
    else ERI_EMB_GRAD(64);
#undef ERI_EMB_GRAD
    if (a.tokens > kFew)
        hipLaunchKernelGGL((embedding_grad_heavy_kernel<TG, TO>), dim3((a.dim + 63) / 64, grid < 32768 ? grid : 32768), dim3(kHeavyThreads), 0, s, a, grid);
}

} // namespace

int launch_embedding(const EriEmbedding &e, uint32_t compute_units, void *stream) {
    const LookupArgs a = {{e.ids, (uint32_t)e.ids_64}, e.table, e.out, (uint32_t)e.tokens, (uint32_t)e.vocab, (uint32_t)e.dim,
                          e.table_stride, e.out_stride, e.scale};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (e.dtype_tag == ERI_DTYPE_F32) launch_lookup_of<float>(a, compute_units, s);
    else launch_lookup_of<bf16>(a, compute_units, s);
    return (int)hipGetLastError();
}

uint64_t embedding_grad_workspace(uint64_t tokens, uint64_t vocab, uint64_t) { return Workspace(tokens, vocab).bytes; }

int launch_embedding_grad(const EriEmbeddingGrad &e, uint32_t, void *stream) {
    const Workspace w(e.tokens, e.vocab);
    char *ws = static_cast<char *>(e.workspace);
    GradArgs a = {{e.ids, (uint32_t)e.ids_64}, e.grad, e.out, (uint32_t *)ws, (Heavy *)(ws + w.heavy), (uint32_t *)(ws + w.first),
                  (uint32_t *)(ws + w.count), (uint32_t)e.tokens, (uint32_t)e.vocab, (uint32_t)e.dim, shift_of(e.vocab), 0,
                  e.grad_stride, e.out_stride, e.padding_id, e.scale, (uint32_t)(e.accumulate != 0)};
    a.locals = (a.vocab + (1u << a.shift) - 1) >> a.shift;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool g32 = e.grad_dtype == ERI_DTYPE_F32, o32 = e.out_dtype == ERI_DTYPE_F32;
    if (g32) o32 ? launch_grad<float, float>(a, s) : launch_grad<float, bf16>(a, s);
    else o32 ? launch_grad<bf16, float>(a, s) : launch_grad<bf16, bf16>(a, s);
    return (int)hipGetLastError();
}

} // namespace eri_layers
