// embedding.hip — rows of a table looked up by token and scaled, and the table's gradient.
//
// The gradient adds up the rows of dout that hold the same token. The tokens are sorted (stably, by the
// radix sort of sort.hpp, on the bits the table's size needs) with their positions, so that a
// token's rows follow each other. A workgroup takes a block of sorted positions, a group of lanes (as many as a row
// has 16-byte vectors) each a run of it, summing in registers; tokens that span runs are joined in LDS,
// tokens that span blocks afterwards from the blocks' partial sums, in order. No float is added
// atomically: the result does not depend on which workgroup runs first. A few tokens take one launch
// instead: every workgroup picks, and sorts, those of its own rows of the table.
#include "internal.hpp"
#include "elem.hpp"
#include "sort.hpp"

namespace tdgs {

constexpr int kEmThreads = 256;
constexpr int kEmBlock = 2048;   // the most sorted positions of a workgroup
constexpr int kEmRun = 32;       // and of one of its runs
constexpr int kEmFew = 4096;         // the most tokens that one launch is taken for, and
constexpr int kEmFewThreads = 512;   // its workgroups' size

struct EmArgs {
    const void *table, *dout, *tokens;
    void *out, *dtable;
    int64_t table_stride, out_stride, dout_stride, dtable_stride, n, vocab, padding, blocks;
    const uint32_t* keys;    // sorted tokens; vocab where there is nothing to add
    const int32_t* order;    // their positions
    float* part;             // 2 rows per block: of the token it begins within, of the token it ends within
    int32_t *list, *count;   // blocks that a token starts in and goes on past; their number
    uint32_t* bad_token;
    float scale;
    int32_t dim, vectors, lanes;   // elements, vectors and lanes per row
    int32_t run, rows, few;        // positions per run; of one launch: table rows per workgroup, tokens (2^k)
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
    // Past the caches: rows written once push out neither the table nor dout's rows, which are read from there (lookup of
    // a million rows of 48 floats 47 -> 33 us, their sums 55 -> 42).
    __device__ __forceinline__ void store(T* __restrict__ p, float scale) const {
        if constexpr (VW == 1) {
            *p = (T)(f[0] * scale);
        } else {
            V v;
#pragma unroll
            for (int i = 0; i < VW; ++i) v[i] = (T)(f[i] * scale);
            __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
        }
    }
};

// Thread per vector of the output. A million rows of 48 floats from 8192: 33 us, 5.8 TB/s of stores.
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
        else atomicOr(a.bad_token, 1u);
        v.store((T*)a.out + row * a.out_stride + e, a.scale);
    }
}

// Sort keys and values: tokens and positions; tokens to leave out sort past the table's end. Also clears
// the `words` that the sort and the list count in, and dtable, whose rows that a token names are written over
// later: that costs less than keeping account of the others (100003 rows of 512 16-bit elements: 17 us, 6 TB/s).
template <class T, int VW>
__global__ __launch_bounds__(kEmThreads) void k_embed_keys(EmArgs a, uint32_t* __restrict__ keys,
                                                           int32_t* __restrict__ values, uint32_t* __restrict__ clear,
                                                           int64_t words, FastDiv by_vectors) {
    const int64_t id = (int64_t)blockIdx.x * kEmThreads + threadIdx.x, step = (int64_t)gridDim.x * kEmThreads;
    for (int64_t i = id; i < a.n; i += step) {
        const int64_t tok = em_token(a, i);
        const bool in = tok >= 0 && tok < a.vocab;
        if (!in) atomicOr(a.bad_token, 1u);
        keys[i] = in && tok != a.padding ? (uint32_t)tok : (uint32_t)a.vocab;
        values[i] = (int32_t)i;
    }
    for (int64_t i = id; i < words; i += step) clear[i] = 0;
    EmVec<T, VW> z;
    z.zero();
    const int64_t total = a.vocab * a.vectors;
    for (int64_t i = id; i < total; i += step) {
        const int64_t row = total <= INT32_MAX ? (int64_t)by_vectors.div((uint32_t)i) : i / a.vectors;
        z.store((T*)a.dtable + row * a.dtable_stride + (i - row * a.vectors) * VW, 0.0f);
    }
}

// Sums a block of sorted positions, `count` of them from LDS (their tokens, and rows of dout): group g of
// the workgroup's lane groups takes `run` of them from g * run on. A token's sum goes to its row of the table;
// that of the token `before` the block, and of one that goes on `after` it, to part (row 0 and row 1).
// Every thread of the workgroup calls it. Returns whether a token starts here and goes on.
template <class T, int VW, int TH, int U, class Row>
__device__ __forceinline__ bool em_block(const EmArgs& a, const uint32_t* s_key, const Row* s_row, int count, int run,
                                         uint32_t before, uint32_t after, float* part, float* s_head, float* s_tail,
                                         uint32_t* s_flag) {
    const int groups = TH / a.lanes, sub = (int)threadIdx.x / a.lanes, col = (int)threadIdx.x % a.lanes;
    const int vec = blockIdx.y * kWave + col, e = vec * VW;
    const bool on = sub < groups && vec < a.vectors;
    const uint32_t none = (uint32_t)a.vocab;
    const int i0 = sub * run, i1 = min(count, i0 + run);
    constexpr uint32_t kHead = 1u, kThrough = 2u, kTail = 4u;
    auto keep = [&](float* s, const EmVec<T, VW>& v) {
#pragma unroll
        for (int i = 0; i < VW; ++i) s[i * TH + threadIdx.x] = v.f[i];
    };
    if (on && i0 < i1) {
        EmVec<T, VW> sum;
        sum.zero();
        uint32_t cur = s_key[i0], flag = 0;
        bool first = cur == (i0 > 0 ? s_key[i0 - 1] : before);
        const uint32_t next = i1 < count ? s_key[i1] : after;
        auto flush = [&](bool last) {
            if (cur == none) return;
            const bool on_past = last && cur == next;
            if (first) {
                keep(s_head, sum);
                flag |= kHead | (on_past ? kThrough : 0u);
            } else if (on_past) {
                keep(s_tail, sum);
                flag |= kTail;
            } else {
                sum.store((T*)a.dtable + (int64_t)cur * a.dtable_stride + e, a.scale);
            }
        };
        for (int i = i0; i < i1; i += U) {
            EmVec<T, VW> v[U];
            uint32_t key[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                key[u] = i + u < i1 ? s_key[i + u] : none;
                v[u].zero();
                if (key[u] != none) v[u].load((const T*)a.dout + (int64_t)s_row[i + u] * a.dout_stride + e);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u < i1 && key[u] != cur) {
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
        if (col == 0) s_flag[sub] = flag;
    } else if (sub < groups && col == 0) {
        s_flag[sub] = 0;
    }
    __syncthreads();
    bool starts = false;
    if (on && i0 < i1) {
        // chains of runs: from a token's start to the run that it ends in, or the block's end
        const uint32_t flag = s_flag[sub];
        auto chain = [&](const float* s, bool through, bool outside) {
            EmVec<T, VW> v;
#pragma unroll
            for (int i = 0; i < VW; ++i) v.f[i] = s[i * TH + threadIdx.x];
            int g = sub + 1;
            for (; through && g < groups && (s_flag[g] & kHead); ++g) {
#pragma unroll
                for (int i = 0; i < VW; ++i) v.f[i] += s_head[i * TH + g * a.lanes + col];
                through = (s_flag[g] & kThrough) != 0;
            }
            const uint32_t key = s_key[i1 - 1];   // (of a tail; a head's that ends here is not stored to its row)
            if (outside || through) {
                float* const p = part + (outside ? 0 : (int64_t)a.vectors * VW) + e;
#pragma unroll
                for (int i = 0; i < VW; ++i) p[i] = v.f[i];
                return !outside;
            }
            v.store((T*)a.dtable + (int64_t)key * a.dtable_stride + e, a.scale);
            return false;
        };
        if (sub == 0 && (flag & kHead)) chain(s_head, (flag & kThrough) != 0, true);
        if (flag & kTail) starts = chain(s_tail, true, false);
    }
    return starts;
}

// A block of sorted positions per workgroup. A million rows of 48 floats: 41 us (192 MB read by position, 4.7 TB/s;
// more rows in flight per thread were no faster).
template <class T, int VW>
__global__ __launch_bounds__(kEmThreads) void k_embed_sums(EmArgs a) {
    __shared__ uint32_t s_key[kEmBlock];
    __shared__ int32_t s_row[kEmBlock];
    __shared__ float s_head[kEmThreads * VW];
    __shared__ float s_tail[kEmThreads * VW];
    __shared__ uint32_t s_flag[kEmThreads];
    const int groups = kEmThreads / a.lanes;
    const uint32_t none = (uint32_t)a.vocab;
    const int size = groups * a.run;
    const int64_t i0 = (int64_t)blockIdx.x * size, i1 = min(a.n, i0 + size);
    for (int i = threadIdx.x; i < (int)(i1 - i0); i += kEmThreads) {
        s_key[i] = a.keys[i0 + i];
        s_row[i] = a.order[i0 + i];
    }
    __syncthreads();
    const bool starts = em_block<T, VW, kEmThreads, (VW == 1 ? 8 : 4), int32_t>(a, s_key, s_row, (int)(i1 - i0), a.run, i0 > 0 ? a.keys[i0 - 1] : none,
                                        i1 < a.n ? a.keys[i1] : none, a.part + 2 * blockIdx.x * ((int64_t)a.vectors * VW),
                                        s_head, s_tail, s_flag);
    if (starts && blockIdx.y == 0 && threadIdx.x % a.lanes == 0) a.list[atomicAdd(a.count, 1)] = (int32_t)blockIdx.x;
}

// A workgroup per token that spans blocks: the end of the block it starts in, then the following blocks'
// beginnings, each lane group adding every so manieth, in order.
template <class T, int VW>
__global__ __launch_bounds__(kEmThreads) void k_embed_join(EmArgs a) {
    __shared__ float s_sum[kEmThreads * VW];
    __shared__ int s_last;
    const int groups = kEmThreads / a.lanes, sub = threadIdx.x / a.lanes;
    const int vec = blockIdx.y * kWave + (int)threadIdx.x % a.lanes, e = vec * VW;
    const bool on = sub < groups && vec < a.vectors;
    const int64_t pitch = (int64_t)a.vectors * VW, size = (int64_t)groups * a.run;
    const int count = *a.count;
    for (int item = blockIdx.x; item < count; item += gridDim.x) {
        const int64_t block = a.list[item];
        const uint32_t key = a.keys[(block + 1) * size];   // (goes on there: the list says so)
        // the last block that begins with the token
        int64_t last = block;
        for (bool more = true; more; ) {
            if (threadIdx.x == 0) s_last = kEmThreads;
            __syncthreads();
            const int64_t r = last + 1 + threadIdx.x;
            if (r >= a.blocks || a.keys[r * size] != key) atomicMin(&s_last, (int)threadIdx.x);
            __syncthreads();
            last += s_last;
            more = s_last == kEmThreads;
            __syncthreads();
        }
        float sum[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) sum[i] = 0.0f;
        if (on) {
#pragma unroll 4
            for (int64_t r = block + sub; r <= last; r += groups) {
                const float* const p = a.part + (2 * r + (r == block ? 1 : 0)) * pitch + e;
#pragma unroll
                for (int i = 0; i < VW; ++i) sum[i] += p[i];
            }
        }
#pragma unroll
        for (int i = 0; i < VW; ++i) s_sum[i * kEmThreads + threadIdx.x] = sum[i];
        __syncthreads();
        if (on && sub == 0) {
            EmVec<T, VW> v;
            v.zero();
            for (int g = 0; g < groups && block + g <= last; ++g)
#pragma unroll
                for (int i = 0; i < VW; ++i) v.f[i] += s_sum[i * kEmThreads + g * a.lanes + (int)threadIdx.x];
            v.store((T*)a.dtable + (int64_t)key * a.dtable_stride + e, a.scale);
        }
        __syncthreads();
    }
}

// One launch for a few tokens: workgroup x takes a.rows <= 4096 rows of the table, picks the tokens that name them,
// sorts them (by token, then position) in LDS, sums, and writes zeros where no token does. Bound by latency: of the tokens,
// five barriers for six bits of the sort, the rows. 96 tokens of 1000: 8 us where the chain of launches takes 31; 2476 of
// 19635, rows of 48 floats: 14 (31); 2600 that are all one token: 23 (23).
template <class T, int VW>
__global__ __launch_bounds__(kEmFewThreads) void k_embed_few(EmArgs a) {
    constexpr int TH = kEmFewThreads, W = TH / kWave, U = 4;
    extern __shared__ uint32_t s_key[];   // keys and rows of a.few tokens each
    __shared__ uint32_t s_other[2 * TH * VW > kEmFew ? 2 * TH * VW : kEmFew];   // the sort's second place, then the sums'
    __shared__ uint32_t s_flag[TH];
    __shared__ int s_wave[U * W], s_digit[64 * W];
    uint16_t* const s_row = (uint16_t*)(s_key + a.few);
    float *const s_head = (float*)s_other, *const s_tail = s_head + TH * VW;
    const int64_t v0 = (int64_t)blockIdx.x * a.rows, v1 = min(a.vocab, v0 + a.rows);
    const int lane = (int)__lane_id(), wave = threadIdx.x / kWave, n = (int)a.n;
    int count = 0;
    for (int i0 = 0; i0 < n; i0 += TH * U) {
        int64_t tok[U];
        uint64_t votes[U];
        int at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) tok[u] = em_token(a, min(i0 + u * TH + (int)threadIdx.x, n - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = i0 + u * TH + (int)threadIdx.x < n;
            if (in && (tok[u] < 0 || tok[u] >= a.vocab) && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(a.bad_token, 1u);
            votes[u] = __ballot(in && tok[u] >= v0 && tok[u] < v1 && tok[u] != a.padding);
            if (lane == 0) s_wave[u * W + wave] = __popcll(votes[u]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w == wave) at[u] = count;
                count += s_wave[u * W + w];
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (votes[u] >> lane & 1) {
                const int p = at[u] + __popcll(votes[u] & lanemask_lt());
                s_key[p] = (uint32_t)(tok[u] - v0) << 12 | (uint32_t)(i0 + u * TH + threadIdx.x);   // (n <= kEmFew = 2^12)
            }
        __syncthreads();
    }
    // sort by token, six bits at a time, each wavefront a piece; positions stay in order
    uint32_t *from = s_key, *to = s_other;
    const int piece = (count + W * kWave - 1) / (W * kWave) * kWave, p0 = wave * piece, p1 = min(count, p0 + piece);
    for (int shift = 12; count > 1 && (a.rows - 1) >> (shift - 12) > 0; shift += 6) {
        auto each = [&](auto&& f) {   // f(key, its digit, the lanes of that digit)
            for (int i = p0; i < p1; i += kWave) {
                const bool in = i + lane < p1;
                const uint32_t key = from[in ? i + lane : i];
                const int digit = (int)(key >> shift & 63u);
                uint64_t same = __ballot(in);
#pragma unroll
                for (int b = 0; b < 6; ++b) {
                    const uint64_t ones = __ballot(digit >> b & 1);
                    same &= digit >> b & 1 ? ones : ~ones;
                }
                if (in) f(key, digit, same);
            }
        };
        int* const mine = s_digit + wave * 64;
        s_digit[threadIdx.x] = 0;
        __syncthreads();
        each([&](uint32_t, int digit, uint64_t same) {
            if ((same & lanemask_lt()) == 0) mine[digit] += __popcll(same);
        });
        __syncthreads();
        // where each digit of each piece goes, digit by digit
        int* const slot = s_digit + (int)threadIdx.x % W * 64 + (int)threadIdx.x / W;
        const int number = *slot;
        int upto = number;
#pragma unroll
        for (int w = 1; w < kWave; w *= 2) {
            const int x = __shfl_up(upto, w, kWave);
            if (lane >= w) upto += x;
        }
        if (lane == kWave - 1) s_wave[wave] = upto;
        __syncthreads();
        for (int w = 0; w < wave; ++w) upto += s_wave[w];
        *slot = upto - number;
        __syncthreads();
        each([&](uint32_t key, int digit, uint64_t same) {
            const int at = mine[digit];
            to[at + __popcll(same & lanemask_lt())] = key;
            if ((same & lanemask_lt()) == 0) mine[digit] = at + __popcll(same);
        });
        __syncthreads();
        uint32_t* const next = from;
        from = to;
        to = next;
    }
    for (int i = threadIdx.x; i < count; i += TH) {
        const uint32_t key = from[i];
        s_row[i] = (uint16_t)(key & 0xfffu);
        s_key[i] = (uint32_t)v0 + (key >> 12);
    }
    __syncthreads();
    const int groups = TH / a.lanes, sub = (int)threadIdx.x / a.lanes;
    const int vec = blockIdx.y * kWave + (int)threadIdx.x % a.lanes;
    const uint32_t none = (uint32_t)a.vocab;
    em_block<T, VW, TH, (VW == 8 ? 8 : 16), uint16_t>(a, s_key, s_row, count, (count + groups - 1) / groups, none, none, nullptr,
                                                      s_head, s_tail, s_flag);
    if (sub >= groups || vec >= a.vectors) return;
    EmVec<T, VW> z;
    z.zero();
    for (int64_t v = v0 + sub; v < v1; v += groups) {
        int lo = 0, hi = count;   // the first place whose token is v or above
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (s_key[mid] < (uint32_t)v) lo = mid + 1;
            else hi = mid;
        }
        if (lo == count || s_key[lo] != (uint32_t)v) z.store((T*)a.dtable + v * a.dtable_stride + vec * VW, 0.0f);
    }
}

// ---- host ----------------------------------------------------------------------------------

static int em_bits(int64_t vocab) {
    int b = 0;
    while ((vocab >> b) != 0) ++b;   // (vocab itself is a key: of the positions left out)
    return b;
}

// Positions per run: kEmRun, fewer where a workgroup would take more than kEmBlock, or where there would
// be less than two workgroups per CU.
static int em_run(int64_t n, int groups) {
    int64_t run = n / (512 * groups);
    if (run > kEmRun) run = kEmRun;
    if (run > kEmBlock / groups) run = kEmBlock / groups;
    return (int)(run > 4 ? run : 4);
}

static int em_lanes(int vectors) { return vectors < kWave ? vectors : kWave; }

// Whether one launch takes n tokens: a thousand, or more where a workgroup has so many lane groups that even if they
// are all one token, a group has 64 rows to add (where that then takes as long as the chain of launches, to 1.5 times that;
// tokens of any spread half of it).
static bool em_few(int64_t n, int groups) {
    const int64_t most = 64 * groups < kEmFew ? 64 * groups : kEmFew;
    return n <= (most > 1024 ? most : 1024);
}

struct EmPlan {
    int vectors, lanes, run;
    bool few;
    int64_t blocks, group_words, clear_words;
    size_t sort_bytes, bytes;
};

static EmPlan em_plan(int64_t n, int64_t vocab, int32_t dim, int vw) {
    EmPlan p = {};
    p.vectors = dim / vw;
    p.lanes = em_lanes(p.vectors);
    p.few = em_few(n, kEmFewThreads / p.lanes);
    if (p.few) return p;
    const int groups = kEmThreads / p.lanes;
    p.run = em_run(n, groups);
    p.blocks = ceil_div(n, (int64_t)groups * p.run);
    p.sort_bytes = radix_temp_bytes(n);
    p.group_words = radix_tiles<uint32_t>(n) <= RsTile<uint32_t>::kGroupedTiles
                        ? radix_group_words<uint32_t>(n, 0, em_bits(vocab)) : 0;
    p.clear_words = p.group_words + 1;   // group sums, the list's count
    ArenaSize s;
    s.take<uint32_t>(p.clear_words);
    for (int i = 0; i < 3; ++i) {
        s.take<uint32_t>(n);
        s.take<int32_t>(n);
    }
    s.take<char>((int64_t)p.sort_bytes);
    s.take<int32_t>(p.blocks);
    s.take<float>(2 * p.blocks * dim);
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
    a.bad_token = ctx_token_word(ctx);
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
    size_t bytes = 0;   // (for whichever vector width the tensors' alignment will allow)
    for (int vw = 1; vw <= 8; vw *= 2) {
        if (dim % vw != 0) break;
        const size_t b = em_plan(n, vocab, dim, vw).bytes;
        if (b > bytes) bytes = b;
    }
    return bytes;
}

int tdgs_embedding_grad(tdgs_ctx* ctx, void* stream_, int32_t dtype, const void* dout, int64_t dout_stride,
                        const void* tokens, int32_t index_bytes, int64_t n, int64_t padding, float scale, void* dtable,
                        int64_t dtable_stride, int64_t vocab, int32_t dim, void* temp, size_t temp_bytes) {
    TDGS_REQUIRE(ctx != nullptr, "embedding: null context");
    TDGS_TRY(em_check(dtype, index_bytes, vocab, dim, n));
    if (vocab == 0) return TDGS_OK;
    TDGS_REQUIRE(padding >= -1 && padding < vocab, "embedding: padding %lld is no row of a table of %lld", (long long)padding,
                 (long long)vocab);
    TDGS_REQUIRE(n == 0 || (tokens && aligned_to(tokens, (size_t)index_bytes)), "embedding: tokens are null or misaligned");
    TDGS_TRY(em_check_rows(dout, "dout", dtype, dout_stride, dim, n, false));
    TDGS_TRY(em_check_rows(dtable, "dtable", dtype, dtable_stride, dim, vocab, true));
    const int vw = em_vw(dtype, dim, dout, dout_stride, dtable, dtable_stride);
    const EmPlan p = em_plan(n, vocab, dim, vw);
    TDGS_REQUIRE(p.bytes == 0 || (temp && temp_bytes >= p.bytes && aligned_to(temp, 16)), "embedding: scratch of %zu bytes, %zu needed",
                 temp ? temp_bytes : (size_t)0, p.bytes);
    hipStream_t stream = (hipStream_t)stream_;
    EmArgs a = {};
    a.dout = dout;
    a.dout_stride = dout_stride;
    a.tokens = tokens;
    a.tokens64 = index_bytes == 8;
    a.dtable = dtable;
    a.dtable_stride = dtable_stride;
    a.n = n;
    a.vocab = vocab;
    a.padding = padding;
    a.scale = scale;
    a.dim = dim;
    a.bad_token = ctx_token_word(ctx);
    a.vectors = p.vectors;
    a.lanes = p.lanes;
    a.run = p.run;
    a.blocks = p.blocks;
    const unsigned column_blocks = (unsigned)ceil_div(a.vectors, kWave);
    if (p.few) {
        // a group of lanes takes a row at a time; two workgroups per CU where the table has the rows, but
        // no more than 2^12 of them in one
        int64_t rows = ceil_div(vocab, 512);
        if (rows < kEmFewThreads / a.lanes) rows = kEmFewThreads / a.lanes;
        if (rows > kEmFew) rows = kEmFew;
        a.rows = (int32_t)rows;
        a.few = 1;
        while (a.few < n) a.few *= 2;
        return em_dispatch(dtype, vw, [&](auto t, auto w) -> int {
            k_embed_few<decltype(t), decltype(w)::value><<<dim3((unsigned)ceil_div(vocab, rows), column_blocks), kEmFewThreads,
                                                           (size_t)a.few * (sizeof(uint32_t) + sizeof(uint16_t)), stream>>>(a);
            TDGS_LAUNCHED();
            return TDGS_OK;
        });
    }
    Arena ar(temp, temp_bytes);
    uint32_t* const clear = ar.take<uint32_t>(p.clear_words);
    uint32_t* k[3];
    int32_t* v[3];
    for (int i = 0; i < 3; ++i) {
        k[i] = ar.take<uint32_t>(n);
        v[i] = ar.take<int32_t>(n);
    }
    void* const sort_temp = ar.take<char>((int64_t)p.sort_bytes);
    a.list = ar.take<int32_t>(p.blocks);
    a.count = (int32_t*)clear + p.group_words;
    a.part = ar.take<float>(2 * p.blocks * dim);
    a.keys = k[1];
    a.order = v[1];
    int64_t key_blocks = ceil_div(n > vocab * a.vectors ? n : vocab * a.vectors, kEmThreads);
    if (key_blocks > 8192) key_blocks = 8192;
    TDGS_TRY(em_dispatch(dtype, vw, [&](auto t, auto w) -> int {
        k_embed_keys<decltype(t), decltype(w)::value><<<(unsigned)key_blocks, kEmThreads, 0, stream>>>(
            a, k[0], v[0], clear, p.clear_words, FastDiv((uint32_t)a.vectors));
        TDGS_LAUNCHED();
        return TDGS_OK;
    }));
    TDGS_TRY(radix_sort_pairs_grouped<uint32_t>(k[0], k[1], v[0], v[1], k[2], v[2], n, 0, em_bits(vocab), sort_temp,
                                                p.sort_bytes, p.group_words > 0 ? clear : nullptr, p.group_words,
                                                stream, ctx_error_word(ctx)));
    return em_dispatch(dtype, vw, [&](auto t, auto w) -> int {
        using T = decltype(t);
        constexpr int VW = decltype(w)::value;
        k_embed_sums<T, VW><<<dim3((unsigned)p.blocks, column_blocks), kEmThreads, 0, stream>>>(a);
        TDGS_LAUNCHED();
        if (p.blocks > 1) {
            k_embed_join<T, VW><<<dim3((unsigned)(p.blocks < 1024 ? p.blocks : 1024), column_blocks), kEmThreads, 0, stream>>>(a);
            TDGS_LAUNCHED();
        }
        return TDGS_OK;
    });
}

}  // extern "C"
