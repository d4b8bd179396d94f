// embedding.hip — rows of a table looked up by token and scaled, and the table's gradient.
//
// The gradient adds up the rows of dout that hold the same token. The tokens are sorted (stably, by the
// radix sort of sort.hpp, on the bits the table's size needs) with their positions, so that a
// token's rows follow each other; runs of kEmRows sorted positions are summed in registers by a few lanes each,
// and a token whose rows lie in several runs is joined afterwards from their partial sums, in order. No
// float is added atomically: the result does not depend on which workgroup runs first.
#include "internal.hpp"
#include "elem.hpp"
#include "sort.hpp"

namespace tdgs {

constexpr int kEmThreads = 256;
constexpr int kEmRows = 32;   // sorted positions per run

struct EmArgs {
    const void *table, *dout, *tokens;
    void *out, *dtable;
    int64_t table_stride, out_stride, dout_stride, dtable_stride, n, vocab, padding, runs;
    const uint32_t* keys;    // sorted tokens; vocab where there is nothing to add
    const int32_t* order;    // their positions
    uint8_t* present;        // whether a token occurs
    float* part;             // 2 rows per run: of the token it begins within, of the token it ends within
    int32_t *list, *count;   // runs that a token starts in and goes on past; their number
    uint32_t* err;
    float scale;
    int32_t dim, vectors, lanes;   // elements, vectors and lanes per row
    bool tokens64;
};

__device__ __forceinline__ int64_t em_token(const EmArgs& a, int64_t i) {
    return a.tokens64 ? ((const int64_t*)a.tokens)[i] : (int64_t)((const int32_t*)a.tokens)[i];
}

template <class T, int VW>
struct EmVec {
    typedef T V __attribute__((ext_vector_type(VW)));
    float f[VW];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < VW; ++i) f[i] = 0.0f;
    }
    __device__ __forceinline__ void load(const T* __restrict__ p) {
        if constexpr (VW == 1) {
            f[0] = (float)*p;
        } else {
            const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
            for (int i = 0; i < VW; ++i) f[i] = (float)v[i];
        }
    }
    __device__ __forceinline__ void store(T* __restrict__ p, float scale) const {
        if constexpr (VW == 1) {
            *p = (T)(f[0] * scale);
        } else {
            V v;
#pragma unroll
            for (int i = 0; i < VW; ++i) v[i] = (T)(f[i] * scale);
            *reinterpret_cast<V*>(p) = v;
        }
    }
};

// Thread per vector of the output.
template <class T, int VW>
__global__ __launch_bounds__(kEmThreads) void k_embed_lookup(EmArgs a, FastDiv by_vectors) {
    const int64_t id0 = (int64_t)blockIdx.x * kEmThreads + threadIdx.x, total = a.n * a.vectors;
    for (int64_t id = id0; id < total; id += (int64_t)gridDim.x * kEmThreads) {
        const int64_t row = total <= INT32_MAX ? (int64_t)by_vectors.div((uint32_t)id) : id / a.vectors;
        const int e = (int)(id - row * a.vectors) * VW;
        const int64_t tok = em_token(a, row);
        EmVec<T, VW> v;
        v.zero();
        if (tok >= 0 && tok < a.vocab) v.load((const T*)a.table + tok * a.table_stride + e);
        else atomicOr(a.err, kErrTokenRange);
        v.store((T*)a.out + row * a.out_stride + e, a.scale);
    }
}

static __global__ __launch_bounds__(kEmThreads) void k_embed_clear(uint32_t* __restrict__ words, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * kEmThreads + threadIdx.x;
    if (i < n) words[i] = 0;
}

// Sort keys and values: tokens and positions; tokens to leave out sort past the table's end.
static __global__ __launch_bounds__(kEmThreads) void k_embed_keys(EmArgs a, uint32_t* __restrict__ keys,
                                                                  int32_t* __restrict__ values) {
    const int64_t i = (int64_t)blockIdx.x * kEmThreads + threadIdx.x;
    if (i >= a.n) return;
    const int64_t tok = em_token(a, i);
    const bool in = tok >= 0 && tok < a.vocab;
    if (!in) atomicOr(a.err, kErrTokenRange);
    const bool use = in && tok != a.padding;
    if (use) a.present[tok] = 1;
    keys[i] = use ? (uint32_t)tok : (uint32_t)a.vocab;
    values[i] = (int32_t)i;
}

// The first workgroups: a few lanes per run of sorted positions, adding its rows token by token; the
// others: rows of the table that no token names become zero.
template <class T, int VW>
__global__ __launch_bounds__(kEmThreads) void k_embed_sums(EmArgs a, int run_blocks) {
    const int lane = (int)__lane_id(), wave = threadIdx.x / kWave;
    const int per_wave = kWave / a.lanes, sub = lane / a.lanes;
    const int vec = blockIdx.y * kWave + lane % a.lanes, e = vec * VW;
    const bool on = sub < per_wave && vec < a.vectors;
    if ((int)blockIdx.x >= run_blocks) {
        const int64_t rows = (int64_t)(gridDim.x - run_blocks) * (kEmThreads / kWave) * per_wave;
        EmVec<T, VW> z;
        z.zero();
        if (on)
            for (int64_t v = ((int64_t)(blockIdx.x - run_blocks) * (kEmThreads / kWave) + wave) * per_wave + sub; v < a.vocab;
                 v += rows)
                if (!a.present[v]) z.store((T*)a.dtable + v * a.dtable_stride + e, 0.0f);
        return;
    }
    const int64_t run = ((int64_t)blockIdx.x * (kEmThreads / kWave) + wave) * per_wave + sub;
    if (!on || run >= a.runs) return;
    const int64_t i0 = run * kEmRows, i1 = min(a.n, i0 + kEmRows);
    const uint32_t none = (uint32_t)a.vocab;
    const uint32_t before = i0 > 0 ? a.keys[i0 - 1] : none, after = i1 < a.n ? a.keys[i1] : none;
    EmVec<T, VW> sum;
    sum.zero();
    uint32_t cur = a.keys[i0];
    bool first = cur == before;   // the run begins within a token
    auto flush = [&](bool last) {
        if (cur == none) return;
        if (first || (last && cur == after)) {
            float* const p = a.part + (2 * run + (first ? 0 : 1)) * ((int64_t)a.vectors * VW) + e;
#pragma unroll
            for (int i = 0; i < VW; ++i) p[i] = sum.f[i];
            if (!first && vec == 0) a.list[atomicAdd(a.count, 1)] = (int32_t)run;
        } else {
            sum.store((T*)a.dtable + (int64_t)cur * a.dtable_stride + e, a.scale);
        }
    };
    constexpr int U = 4;
    for (int64_t i = i0; i < i1; i += U) {
        EmVec<T, VW> v[U];
        uint32_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = i + u < i1;
            key[u] = in ? a.keys[i + u] : none;
            v[u].zero();
            if (key[u] != none) v[u].load((const T*)a.dout + (int64_t)a.order[i + u] * a.dout_stride + e);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= i1) break;
            if (key[u] != cur) {
                flush(false);
                cur = key[u];
                first = false;
                sum.zero();
            }
#pragma unroll
            for (int k = 0; k < VW; ++k) sum.f[k] += v[u].f[k];
        }
    }
    flush(true);
}

// A workgroup per token that spans runs: the end of the run it starts in, then the following runs'
// beginnings, each lane group adding every so manieth, in order.
template <class T, int VW>
__global__ __launch_bounds__(kEmThreads) void k_embed_join(EmArgs a) {
    __shared__ float s_sum[kEmThreads * VW];
    __shared__ int s_last;
    const int groups = kEmThreads / a.lanes, sub = threadIdx.x / a.lanes;
    const int vec = blockIdx.y * kWave + (int)threadIdx.x % a.lanes, e = vec * VW;
    const bool on = sub < groups && vec < a.vectors;
    const int64_t pitch = (int64_t)a.vectors * VW;
    const int count = *a.count;
    for (int item = blockIdx.x; item < count; item += gridDim.x) {
        const int64_t run = a.list[item];
        const uint32_t key = a.keys[(run + 1) * kEmRows];   // (goes on there: the list says so)
        // the last run that begins with the token
        int64_t last = run;
        for (bool more = true; more; ) {
            if (threadIdx.x == 0) s_last = kEmThreads;
            __syncthreads();
            const int64_t r = last + 1 + threadIdx.x;
            if (r >= a.runs || a.keys[r * kEmRows] != key) atomicMin(&s_last, (int)threadIdx.x);
            __syncthreads();
            last += s_last;
            more = s_last == kEmThreads;
            __syncthreads();
        }
        float sum[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) sum[i] = 0.0f;
        if (on)
            for (int64_t r = run + sub; r <= last; r += groups) {
                const float* const p = a.part + (2 * r + (r == run ? 1 : 0)) * pitch + e;
#pragma unroll
                for (int i = 0; i < VW; ++i) sum[i] += p[i];
            }
#pragma unroll
        for (int i = 0; i < VW; ++i) s_sum[threadIdx.x * VW + i] = sum[i];
        __syncthreads();
        if (on && sub == 0) {
            EmVec<T, VW> v;
            v.zero();
            for (int g = 0; g < groups && run + g <= last; ++g)
#pragma unroll
                for (int i = 0; i < VW; ++i) v.f[i] += s_sum[(g * a.lanes + (int)threadIdx.x) * VW + i];
            v.store((T*)a.dtable + (int64_t)key * a.dtable_stride + e, a.scale);
        }
        __syncthreads();
    }
}

// ---- host ----------------------------------------------------------------------------------

static int em_bits(int64_t vocab) {
    int b = 0;
    while ((vocab >> b) != 0) ++b;   // (vocab itself is a key: of the positions left out)
    return b;
}

static int64_t em_runs(int64_t n) { return ceil_div(n, kEmRows); }

struct EmPlan {
    int64_t runs, group_words, clear_words;
    size_t sort_bytes, bytes;
};

static EmPlan em_plan(int64_t n, int64_t vocab, int32_t dim) {
    EmPlan p;
    p.runs = em_runs(n);
    p.sort_bytes = radix_temp_bytes(n);
    p.group_words = radix_tiles<uint32_t>(n) <= RsTile<uint32_t>::kGroupedTiles
                        ? radix_group_words<uint32_t>(n, 0, em_bits(vocab)) : 0;
    p.clear_words = p.group_words + 1 + ceil_div(vocab, 4);   // group sums, the list's count, present
    ArenaSize s;
    s.take<uint32_t>(p.clear_words);
    for (int i = 0; i < 3; ++i) {
        s.take<uint32_t>(n);
        s.take<int32_t>(n);
    }
    s.take<char>((int64_t)p.sort_bytes);
    s.take<int32_t>(p.runs);
    s.take<float>(2 * p.runs * dim);
    p.bytes = s.used;
    return p;
}

static int em_check(int32_t dtype, int32_t index_bytes, int64_t vocab, int32_t dim, int64_t n) {
    TDGS_REQUIRE(known_dtype(dtype), "embedding: unknown element type %d", dtype);
    TDGS_REQUIRE(index_bytes == 4 || index_bytes == 8, "embedding: tokens of %d bytes, not 4 or 8", index_bytes);
    TDGS_REQUIRE(vocab >= 0 && vocab < INT32_MAX && dim > 0 && dim <= (1 << 20), "embedding: table of %lld rows of %d",
                 (long long)vocab, dim);
    TDGS_REQUIRE(n >= 0 && n < INT32_MAX, "embedding: %lld tokens", (long long)n);
    return TDGS_OK;
}

static int em_vw(int32_t dtype, int32_t dim, const void* p, int64_t ps, const void* q, int64_t qs) {
    const int64_t e = dtype_size(dtype);
    return dim * e % 16 == 0 && aligned_to(p, 16) && aligned_to(q, 16) && ps * e % 16 == 0 && qs * e % 16 == 0
               ? (int)(16 / e) : 1;
}

static int em_check_rows(const void* p, const char* name, int32_t dtype, int64_t stride, int32_t dim, int64_t n, bool written) {
    if (n == 0) return TDGS_OK;
    TDGS_REQUIRE(p != nullptr, "embedding: %s is null", name);
    TDGS_REQUIRE(aligned_to(p, (size_t)dtype_size(dtype)), "embedding: %s is not aligned to its element type", name);
    TDGS_REQUIRE(stride >= (written && n > 1 ? dim : 0), "embedding: rows of %s overlap", name);
    return TDGS_OK;
}

// f(T{}, vector width)
template <class F>
static int em_dispatch(int32_t dtype, int vw, F&& f) {
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        return vw == 1 ? f(t, std::integral_constant<int, 1>{}) : f(t, std::integral_constant<int, 16 / (int)sizeof(T)>{});
    });
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

int tdgs_embedding_lookup(tdgs_ctx* ctx, void* stream_, int32_t dtype, const void* table, int64_t table_stride,
                          int64_t vocab, int32_t dim, const void* tokens, int32_t index_bytes, int64_t n, float scale,
                          void* out, int64_t out_stride) {
    TDGS_REQUIRE(ctx != nullptr, "embedding: null context");
    TDGS_TRY(em_check(dtype, index_bytes, vocab, dim, n));
    if (n == 0) return TDGS_OK;
    TDGS_REQUIRE(tokens && aligned_to(tokens, (size_t)index_bytes), "embedding: tokens are null or misaligned");
    TDGS_TRY(em_check_rows(table, "table", dtype, table_stride, dim, vocab, false));
    TDGS_TRY(em_check_rows(out, "out", dtype, out_stride, dim, n, true));
    EmArgs a = {};
    a.table = table;
    a.table_stride = table_stride;
    a.tokens = tokens;
    a.tokens64 = index_bytes == 8;
    a.out = out;
    a.out_stride = out_stride;
    a.n = n;
    a.vocab = vocab;
    a.scale = scale;
    a.dim = dim;
    a.err = ctx_error_word(ctx);
    const int vw = em_vw(dtype, dim, table, table_stride, out, out_stride);
    a.vectors = dim / vw;
    int64_t blocks = ceil_div(n * a.vectors, kEmThreads);
    if (blocks > 65536) blocks = 65536;
    hipStream_t stream = (hipStream_t)stream_;
    return em_dispatch(dtype, vw, [&](auto t, auto w) -> int {
        k_embed_lookup<decltype(t), decltype(w)::value>
            <<<(unsigned)blocks, kEmThreads, 0, stream>>>(a, FastDiv((uint32_t)a.vectors));
        TDGS_LAUNCHED();
        return TDGS_OK;
    });
}

size_t tdgs_embedding_grad_temp_bytes(int64_t n, int64_t vocab, int32_t dim) {
    if (em_check(TDGS_F32, 4, vocab, dim, n) != TDGS_OK) return 0;
    return em_plan(n, vocab, dim).bytes;
}

int tdgs_embedding_grad(tdgs_ctx* ctx, void* stream_, int32_t dtype, const void* dout, int64_t dout_stride,
                        const void* tokens, int32_t index_bytes, int64_t n, int64_t padding, float scale, void* dtable,
                        int64_t dtable_stride, int64_t vocab, int32_t dim, void* temp, size_t temp_bytes) {
    TDGS_REQUIRE(ctx != nullptr, "embedding: null context");
    TDGS_TRY(em_check(dtype, index_bytes, vocab, dim, n));
    if (vocab == 0) return TDGS_OK;
    TDGS_REQUIRE(n == 0 || (tokens && aligned_to(tokens, (size_t)index_bytes)), "embedding: tokens are null or misaligned");
    TDGS_TRY(em_check_rows(dout, "dout", dtype, dout_stride, dim, n, false));
    TDGS_TRY(em_check_rows(dtable, "dtable", dtype, dtable_stride, dim, vocab, true));
    const EmPlan p = em_plan(n, vocab, dim);
    TDGS_REQUIRE(temp && temp_bytes >= p.bytes && aligned_to(temp, 16), "embedding: scratch of %zu bytes, %zu needed",
                 temp ? temp_bytes : (size_t)0, p.bytes);
    hipStream_t stream = (hipStream_t)stream_;
    Arena ar(temp, temp_bytes);
    EmArgs a = {};
    uint32_t* const clear = ar.take<uint32_t>(p.clear_words);
    uint32_t* k[3];
    int32_t* v[3];
    for (int i = 0; i < 3; ++i) {
        k[i] = ar.take<uint32_t>(n);
        v[i] = ar.take<int32_t>(n);
    }
    void* const sort_temp = ar.take<char>((int64_t)p.sort_bytes);
    a.list = ar.take<int32_t>(p.runs);
    a.count = (int32_t*)clear + p.group_words;
    a.part = ar.take<float>(2 * p.runs * dim);
    a.present = (uint8_t*)(clear + p.group_words + 1);
    a.dout = dout;
    a.dout_stride = dout_stride;
    a.tokens = tokens;
    a.tokens64 = index_bytes == 8;
    a.dtable = dtable;
    a.dtable_stride = dtable_stride;
    a.n = n;
    a.vocab = vocab;
    a.padding = padding;
    a.runs = p.runs;
    a.scale = scale;
    a.dim = dim;
    a.err = ctx_error_word(ctx);
    const int vw = em_vw(dtype, dim, dout, dout_stride, dtable, dtable_stride);
    a.vectors = dim / vw;
    a.lanes = a.vectors < kWave ? a.vectors : kWave;
    a.keys = k[1];
    a.order = v[1];
    k_embed_clear<<<(unsigned)ceil_div(p.clear_words, kEmThreads), kEmThreads, 0, stream>>>(clear, p.clear_words);
    TDGS_LAUNCHED();
    if (n > 0) {
        k_embed_keys<<<(unsigned)ceil_div(n, kEmThreads), kEmThreads, 0, stream>>>(a, k[0], v[0]);
        TDGS_LAUNCHED();
        TDGS_TRY(radix_sort_pairs_grouped<uint32_t>(k[0], k[1], v[0], v[1], k[2], v[2], n, 0, em_bits(vocab), sort_temp,
                                                    p.sort_bytes, p.group_words > 0 ? clear : nullptr, p.group_words,
                                                    stream, a.err));
    }
    const int per_block = kEmThreads / kWave * (kWave / a.lanes);
    const int64_t run_blocks = ceil_div(p.runs, per_block);
    int64_t zero_blocks = ceil_div(vocab, per_block);
    if (zero_blocks > 2048) zero_blocks = 2048;
    const unsigned column_blocks = (unsigned)ceil_div(a.vectors, kWave);
    return em_dispatch(dtype, vw, [&](auto t, auto w) -> int {
        using T = decltype(t);
        constexpr int VW = decltype(w)::value;
        k_embed_sums<T, VW><<<dim3((unsigned)(run_blocks + zero_blocks), column_blocks), kEmThreads, 0, stream>>>(
            a, (int)run_blocks);
        TDGS_LAUNCHED();
        if (p.runs > 1) {
            k_embed_join<T, VW><<<dim3((unsigned)(p.runs < 1024 ? p.runs : 1024), column_blocks), kEmThreads, 0, stream>>>(a);
            TDGS_LAUNCHED();
        }
        return TDGS_OK;
    });
}

}  // extern "C"
