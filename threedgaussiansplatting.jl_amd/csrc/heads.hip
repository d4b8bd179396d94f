// heads.hip — norms of queries and keys for each head with their rotation by position on several axes in the
// same pass, and its gradient.
//
// A head's row of d elements is split into units of V pairs, one per lane: V elements of each half (pairs p,
// p + pairs), or 2 V neighbours (pairs 2 p, 2 p + 1, and what is not rotated), so that both elements of a pair
// are in one lane and the norm's sum takes a few exchanges among the row's lanes; a wavefront takes as many whole rows as it
// has lanes for. A workgroup takes a few tokens at a time: it makes their cosines and sines, and the places of their
// rows, once, in LDS, and uses them for all heads, of the queries first and then of the keys, whose weights
// stay in registers.
//
// The angle of a far position has few bits left in 32: position * frequency / (2 pi) is taken in 64 bits, as turns,
// whose whole part is dropped; the rest is exact to 2^-26 in 32 bits, from which sinpi and cospi go on.
//
// With r = 1 / sqrt(mean x^2 + eps), xhat = r x, u the output's gradient rotated back and e = u w:
// dw = sum u xhat, dx = r (e - xhat mean(e xhat)); r is computed again from x, which is read anyway. All of it is
// bound by memory: each row is read once and written once. 32400 tokens x 32 heads of 64 bfloat16: 60 us (265 MB, 4.4 TB/s),
// the rotation alone 57, gradients 85; few tokens by the latency of their positions, rows and stores.
#include "internal.hpp"
#include "elem.hpp"
#include "overlap.hpp"

namespace tdgs {

constexpr int kHnThreads = 256;
constexpr int kHnAngles = 4096;     // of a workgroup's tokens, in LDS: 32 KB
constexpr int kHnBlocks = 1024;     // workgroups of the gradient, which leave one partial sum of dw each
constexpr int kHnMostBlocks = 1 << 23;   // of any launch, which has fewer than 2^32 threads
constexpr int kHnMaxDim = 256;
constexpr int kHnTokens = 64;       // of a workgroup at a time, at most

struct HnTensor {
    const void *x, *dout;
    void* out;                       // y, or dx
    int64_t xb, xl, xh, db, dl, dh, ob, ol, oh;
    const void* weight;
};

struct HnArgs {
    HnTensor t[2];                   // queries, keys
    const double* turns;
    const void* positions;
    int64_t position_batch, tokens;  // tokens: batch * length
    float* part;
    int32_t length, heads[2], d, pairs, axes;
    int32_t ends[4];                 // pairs of the axes up to and with this one
    int32_t position_type, per;      // per: tokens at a time
    int32_t lanes, units, rotated_units;   // lanes of a row, with one unit each or (N = 2) two
    float eps, inv_d, sign;
    bool norm, interleaved, param_f32;
    FastDiv by_heads[2], by_length, by_pairs;
};

__device__ __forceinline__ double hn_position(const HnArgs& a, int64_t i) {
    switch (a.position_type) {
        case TDGS_POSITION_I32: return (double)((const int32_t*)a.positions)[i];
        case TDGS_POSITION_I64: return (double)((const int64_t*)a.positions)[i];
        default: return (double)((const float*)a.positions)[i];
    }
}

// Where the rows of the tokens at hand start: x, output, output's gradient; of queries and keys.
struct HnPlaces {
    int64_t x[2][kHnTokens], out[2][kHnTokens], dout[2][kHnTokens];
};

// The places of `count` tokens from `first` on, and cosine and sine of their pairs.
template <bool GRAD>
__device__ __forceinline__ void hn_tokens(const HnArgs& a, int64_t first, int count, HnPlaces& at, float2* s) {
    // (arguments are indexed by constants: a lane's own index would load them from memory, one wait after the other)
    for (int token = threadIdx.x; token < count; token += kHnThreads) {
        const uint32_t row = (uint32_t)(first + token), b = a.by_length.div(row), l = row - b * a.by_length.d;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const HnTensor& t = a.t[k];
            at.x[k][token] = b * t.xb + l * t.xl;
            at.out[k][token] = b * t.ob + l * t.ol;
            if (GRAD) at.dout[k][token] = b * t.db + l * t.dl;
        }
    }
    for (int i = threadIdx.x; i < count * a.pairs; i += kHnThreads) {
        const int token = (int)a.by_pairs.div((uint32_t)i), p = i - token * a.pairs;
        const uint32_t row = (uint32_t)(first + token), b = a.by_length.div(row), l = row - b * a.by_length.d;
        const int axis = (p >= a.ends[0]) + (p >= a.ends[1]) + (p >= a.ends[2]);   // (unused axes end with the last one)
        const double t = hn_position(a, b * a.position_batch + (int64_t)l * a.axes + axis) * a.turns[p];
        float sn, cs;
        sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
        s[i] = make_float2(cs, a.sign * sn);
    }
}

// What the units of a call are: elements of both halves all, neighbours all (interleaved pairs, or none rotated), or
// halves with a rest that is not rotated.
enum { kHnHalves, kHnNeighbours, kHnMixed };

// The two sets of V elements of unit j of a row: where they start, how far elements of a set are apart and whether they
// are rotated. ALL: there is a unit for every lane.
template <int V, int KIND, bool ALL>
struct HnUnit {
    int first, second, step, pair;
    bool on, rotated;
    __device__ __forceinline__ HnUnit(const HnArgs& a, int j) {
        on = ALL || j < a.units;
        rotated = KIND == kHnHalves || j < a.rotated_units;
        pair = j * V;
        if (KIND == kHnHalves || (KIND == kHnMixed && rotated)) {
            first = j * V;
            second = a.pairs + j * V;
            step = 1;
        } else {
            first = rotated ? 2 * j * V : 2 * a.pairs + 2 * (j - a.rotated_units) * V;
            second = first + 1;
            step = 2;
        }
    }
};

// A unit's 2 V elements at p, as V first and V second ones of its pairs.
template <class T, int V, int KIND, bool ALL>
__device__ __forceinline__ void hn_load(const T* __restrict__ p, const HnUnit<V, KIND, ALL>& u, int d, float (&a)[V], float (&b)[V]) {
    if constexpr (V == 1) {
        a[0] = u.on ? (float)p[u.first] : 0.0f;
        b[0] = u.on && u.second < d ? (float)p[u.second] : 0.0f;
    } else {
        typedef T W __attribute__((ext_vector_type(V)));
        typedef T Wa __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        const bool halves = KIND == kHnHalves || (KIND == kHnMixed && u.step == 1);
        const W x = *reinterpret_cast<const Wa*>(p + u.first);
        const W y = *reinterpret_cast<const Wa*>(p + (halves ? u.second : u.first + V));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // neighbours: element 2 i and 2 i + 1 of the 2 V
            const T even = 2 * i < V ? x[2 * i % V] : y[2 * i % V], odd = 2 * i < V ? x[(2 * i + 1) % V] : y[(2 * i + 1) % V];
            a[i] = (float)(halves ? x[i] : even);
            b[i] = (float)(halves ? y[i] : odd);
        }
    }
}

template <class T, int V, int KIND, bool ALL>
__device__ __forceinline__ void hn_store(T* __restrict__ p, const HnUnit<V, KIND, ALL>& u, int d, const float (&a)[V],
                                         const float (&b)[V]) {
    if (!u.on) return;
    if constexpr (V == 1) {
        p[u.first] = (T)a[0];
        if (u.second < d) p[u.second] = (T)b[0];
    } else {
        typedef T W __attribute__((ext_vector_type(V)));
        typedef T Wa __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        const bool halves = KIND == kHnHalves || (KIND == kHnMixed && u.step == 1);
        W x, y;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float lo = i % 2 ? b[i / 2] : a[i / 2], hi = i % 2 ? b[(V + i) / 2] : a[(V + i) / 2];
            x[i] = (T)(halves ? a[i] : lo);
            y[i] = (T)(halves ? b[i] : hi);
        }
        *reinterpret_cast<Wa*>(p + u.first) = x;
        *reinterpret_cast<Wa*>(p + (halves ? u.second : u.first + V)) = y;
    }
}

// A lane's weights, of queries and of keys: they stay in registers. All of them are loaded at once, from elements that exist (one
// load behind a branch after the other took a workgroup longer than its rows).
template <class T, int V, int N, int KIND>
struct HnWeights {
    float x[2][N][V], y[2][N][V];
    template <class W>
    __device__ __forceinline__ void load(const W* w, const HnArgs& a, int k, int lane) {
        W first[N][V], second[N][V];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const HnUnit<V, KIND, N == 1> u(a, lane + n * a.lanes);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int f = u.first + i * u.step, s = u.second + i * u.step;
                first[n][i] = w[f < a.d ? f : a.d - 1];
                second[n][i] = w[s < a.d ? s : a.d - 1];
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[k][n][i] = (float)first[n][i];
                y[k][n][i] = (float)second[n][i];
            }
    }
    __device__ __forceinline__ HnWeights(const HnArgs& a, int lane) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const void* const w = a.t[k].weight;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < V; ++i) x[k][n][i] = y[k][n][i] = 1.0f;
            if (w && a.param_f32) load((const float*)w, a, k, lane);
            else if (w) load((const T*)w, a, k, lane);
        }
    }
};

// The sum of a row's lanes, of which this is lane j of `lanes` neighbours, in all of them.
__device__ __forceinline__ float hn_row_sum(float x, int j, int lanes) {
    if ((lanes & (lanes - 1)) == 0) {
        for (int w = lanes >> 1; w > 0; w >>= 1) x += __shfl_xor(x, w, kWave);
        return x;
    }
    const int me = (int)__lane_id();
    for (int w = 1; w < lanes; w <<= 1) {   // lane j then holds those from j up to j + 2 w
        const float y = __shfl(x, me + w, kWave);
        x += j + w < lanes ? y : 0.0f;
    }
    return __shfl(x, me - j, kWave);
}

// (a, b) turned by the angles of s; by the opposite ones with BACK.
template <int V, bool BACK>
__device__ __forceinline__ void hn_turn(const float2* s, float (&a)[V], float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 cs = s[i];
        const float sn = BACK ? -cs.y : cs.y, x = a[i], y = b[i];
        a[i] = __builtin_fmaf(x, cs.x, -(y * sn));
        b[i] = __builtin_fmaf(x, sn, y * cs.x);
    }
}

// A thread's place: unit j of the sub-th of the rows that a workgroup takes at once.
struct HnLane {
    int j, sub, rows;
    bool on;
    __device__ __forceinline__ HnLane(const HnArgs& a) {
        const int lane = (int)__lane_id(), per = kWave / a.lanes, row = lane / a.lanes;
        j = lane - row * a.lanes;
        on = row < per;
        sub = (int)threadIdx.x / kWave * per + (on ? row : 0);
        rows = kHnThreads / kWave * per;
    }
};

// N units per lane (two where a head of more than 128 elements goes by single pairs).
template <class T, int V, int N, int KIND>
__global__ __launch_bounds__(kHnThreads) void k_head_norm(HnArgs a) {
    constexpr int U = 4;
    extern __shared__ float2 s_angles[];
    __shared__ HnPlaces s_at;
    const HnLane lane(a);
    const HnWeights<T, V, N, KIND> w(a, lane.j);
    for (int64_t first = (int64_t)blockIdx.x * a.per; first < a.tokens; first += (int64_t)gridDim.x * a.per) {
        const int count = (int)(a.tokens - first < a.per ? a.tokens - first : a.per);
        __syncthreads();   // (the tokens before)
        hn_tokens<false>(a, first, count, s_at, s_angles);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const HnTensor& t = a.t[k];
            const int rows = count * a.heads[k];
            // U rows at once, for their loads (every lane stays for the sums)
            for (int r0 = 0; r0 < rows; r0 += U * lane.rows) {
                float ya[U][N][V], yb[U][N][V];
                int token[U], head[U];
#pragma unroll
                for (int m = 0; m < U; ++m) {
                    const int at = r0 + m * lane.rows + lane.sub, r = at < rows ? at : rows - 1;
                    token[m] = (int)a.by_heads[k].div((uint32_t)r);
                    head[m] = r - token[m] * a.heads[k];
                    const T* const x = (const T*)t.x + s_at.x[k][token[m]] + head[m] * t.xh;
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        hn_load<T>(x, HnUnit<V, KIND, N == 1>(a, lane.j + n * a.lanes), a.d, ya[m][n], yb[m][n]);
                }
#pragma unroll
                for (int m = 0; m < U; ++m) {
                    if (m > 0 && r0 + m * lane.rows >= rows) break;
                    if (a.norm) {
                        float sum = 0.0f;
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int i = 0; i < V; ++i)
                                sum = __builtin_fmaf(ya[m][n][i], ya[m][n][i], __builtin_fmaf(yb[m][n][i], yb[m][n][i], sum));
                        sum = rsqrtf(__builtin_fmaf(hn_row_sum(sum, lane.j, a.lanes), a.inv_d, a.eps));
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                ya[m][n][i] *= sum * w.x[k][n][i];
                                yb[m][n][i] *= sum * w.y[k][n][i];
                            }
                    }
                    T* const out = (T*)t.out + s_at.out[k][token[m]] + head[m] * t.oh;
                    const bool valid = lane.on && r0 + m * lane.rows + lane.sub < rows;
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const HnUnit<V, KIND, N == 1> u(a, lane.j + n * a.lanes);
                        if (u.on && u.rotated) hn_turn<V, false>(s_angles + token[m] * a.pairs + u.pair, ya[m][n], yb[m][n]);
                        if (valid) hn_store<T>(out, u, a.d, ya[m][n], yb[m][n]);
                    }
                }
            }
        }
    }
}

// dx, and this workgroup's sums for dw: part[block][queries, keys][d].
template <class T, int V, int N, int KIND>
__global__ __launch_bounds__(kHnThreads) void k_head_norm_grad(HnArgs a) {
    extern __shared__ float2 s_angles[];
    __shared__ HnPlaces s_at;
    const HnLane lane(a);
    const HnWeights<T, V, N, KIND> w(a, lane.j);
    float da[2][N][V], db[2][N][V];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < V; ++i) da[k][n][i] = db[k][n][i] = 0.0f;
    for (int64_t first = (int64_t)blockIdx.x * a.per; first < a.tokens; first += (int64_t)gridDim.x * a.per) {
        const int count = (int)(a.tokens - first < a.per ? a.tokens - first : a.per);
        __syncthreads();
        hn_tokens<true>(a, first, count, s_at, s_angles);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const HnTensor& t = a.t[k];
            const int rows = count * a.heads[k];
            for (int r0 = 0; r0 < rows; r0 += lane.rows) {
                const bool valid = lane.on && r0 + lane.sub < rows;
                const int row = r0 + lane.sub < rows ? r0 + lane.sub : rows - 1;
                const int token = (int)a.by_heads[k].div((uint32_t)row), head = row - token * a.heads[k];
                const T* const x = (const T*)t.x + s_at.x[k][token] + head * t.xh;
                const T* const dout = (const T*)t.dout + s_at.dout[k][token] + head * t.dh;
                float xa[N][V], xb[N][V], ea[N][V], eb[N][V], sum = 0.0f, mean = 0.0f;
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const HnUnit<V, KIND, N == 1> u(a, lane.j + n * a.lanes);
                    hn_load<T>(x, u, a.d, xa[n], xb[n]);
                    hn_load<T>(dout, u, a.d, ea[n], eb[n]);
                }
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < V; ++i) sum = __builtin_fmaf(xa[n][i], xa[n][i], __builtin_fmaf(xb[n][i], xb[n][i], sum));
                const float r = rsqrtf(__builtin_fmaf(hn_row_sum(sum, lane.j, a.lanes), a.inv_d, a.eps));
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const HnUnit<V, KIND, N == 1> u(a, lane.j + n * a.lanes);
                    if (u.on && u.rotated) hn_turn<V, true>(s_angles + token * a.pairs + u.pair, ea[n], eb[n]);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        xa[n][i] *= r;
                        xb[n][i] *= r;
                        const float pa = ea[n][i] * xa[n][i], pb = eb[n][i] * xb[n][i];
                        da[k][n][i] += valid ? pa : 0.0f;
                        db[k][n][i] += valid ? pb : 0.0f;
                        mean = __builtin_fmaf(pa, w.x[k][n][i], __builtin_fmaf(pb, w.y[k][n][i], mean));
                    }
                }
                mean = hn_row_sum(mean, lane.j, a.lanes) * a.inv_d;
                T* const out = (T*)t.out + s_at.out[k][token] + head * t.oh;
#pragma unroll
                for (int n = 0; n < N; ++n) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        xa[n][i] = r * __builtin_fmaf(-mean, xa[n][i], ea[n][i] * w.x[k][n][i]);
                        xb[n][i] = r * __builtin_fmaf(-mean, xb[n][i], eb[n][i] * w.y[k][n][i]);
                    }
                    if (valid) hn_store<T>(out, HnUnit<V, KIND, N == 1>(a, lane.j + n * a.lanes), a.d, xa[n], xb[n]);
                }
            }
        }
    }
    if (!a.part) return;
    // over the rows that were taken at once: every thread's 2 N V elements
    __shared__ float s_sums[kHnThreads * 2 * V * N];
    const int across = kHnThreads / a.d, y = (int)threadIdx.x / a.d, c = (int)threadIdx.x - y * a.d;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float* const part = a.part + ((int64_t)blockIdx.x * 2 + k) * a.d;
        if (a.heads[k] == 0) {
            if (y == 0) part[c] = 0.0f;
            continue;
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const HnUnit<V, KIND, N == 1> u(a, lane.j + n * a.lanes);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!lane.on || !u.on) continue;
                s_sums[lane.sub * a.d + u.first + i * u.step] = da[k][n][i];
                if (u.second + i * u.step < a.d) s_sums[lane.sub * a.d + u.second + i * u.step] = db[k][n][i];
            }
        }
        // a column by as many threads as there are for it, up to eight rows each, whose sums are joined in turn or, if they are
        // many, by halves: all rows one after the other, the 128 of heads of 16 left twice the error
        float x = 0.0f;
        __syncthreads();
        if (y < across)
            for (int r = y; r < lane.rows; r += across) x += s_sums[r * a.d + c];
        __syncthreads();
        if (y < across) s_sums[threadIdx.x] = x;
        int left = across;
        for (; left > 8; left = (left + 1) / 2) {
            __syncthreads();
            const int half = (left + 1) / 2;
            if (y < left - half) s_sums[threadIdx.x] += s_sums[threadIdx.x + half * a.d];
        }
        __syncthreads();
        if (y == 0) {
            x = s_sums[c];
            for (int i = 1; i < left; ++i) x += s_sums[i * a.d + c];
            part[c] = x;
        }
    }
}

// Column c of part's 2 d, its blocks shared out over 32 lanes.
constexpr int kHnJoinCols = 8;
template <class T>
__global__ __launch_bounds__(kHnThreads) void k_head_norm_join(const float* __restrict__ part, int blocks, int d, void* dq, void* dk,
                                                               bool f32) {
    __shared__ float s[kHnThreads / kHnJoinCols][kHnJoinCols + 1];
    const int c = blockIdx.x * kHnJoinCols + (int)threadIdx.x % kHnJoinCols, y = (int)threadIdx.x / kHnJoinCols;
    float x = 0.0f;
    if (c < 2 * d) {
#pragma unroll 8
        for (int b = y; b < blocks; b += kHnThreads / kHnJoinCols) x += part[(int64_t)b * 2 * d + c];
    }
    s[y][threadIdx.x % kHnJoinCols] = x;
    for (int w = kHnThreads / kHnJoinCols / 2; w > 0; w >>= 1) {
        __syncthreads();
        if (y < w) s[y][threadIdx.x % kHnJoinCols] += s[y + w][threadIdx.x % kHnJoinCols];
    }
    if (y != 0 || c >= 2 * d) return;
    x = s[0][threadIdx.x];
    void* const p = c < d ? dq : dk;
    if (!p) return;
    const int e = c < d ? c : c - d;
    if (f32) ((float*)p)[e] = x;
    else ((T*)p)[e] = (T)x;
}

// ---- host ----------------------------------------------------------------------------------

static int hn_check(const tdgs_head_norm* a) {
    TDGS_REQUIRE(a != nullptr, "head norm: null arguments");
    TDGS_REQUIRE(known_dtype(a->dtype), "head norm: unknown element type %d", a->dtype);
    TDGS_REQUIRE(a->param_dtype == a->dtype || a->param_dtype == TDGS_F32,
                 "head norm: weights must be float32 or of the input's type");
    TDGS_REQUIRE(aligned_to(a->q_weight, (size_t)dtype_size(a->param_dtype)) && aligned_to(a->k_weight, (size_t)dtype_size(a->param_dtype)),
                 "head norm: the weights are not aligned to their element type");
    TDGS_REQUIRE(a->batch >= 0 && a->length >= 0 && a->heads >= 0 && a->kv_heads >= 0, "head norm: negative size");
    TDGS_REQUIRE(a->heads <= 65536 && a->kv_heads <= 65536, "head norm: %d and %d heads", a->heads, a->kv_heads);
    TDGS_REQUIRE((int64_t)a->batch * a->length <= INT32_MAX - 65536, "head norm: too many tokens");
    TDGS_REQUIRE(a->head_dim >= 1 && a->head_dim <= kHnMaxDim, "head norm: head dimension %d is not in 1 to %d", a->head_dim,
                 kHnMaxDim);
    TDGS_REQUIRE(a->eps >= 0.0f && a->eps < INFINITY, "head norm: eps must be finite and not negative");
    TDGS_REQUIRE(a->pairs >= 0 && 2 * (int64_t)a->pairs <= a->head_dim, "head norm: %d rotated pairs in a head of %d", a->pairs,
                 a->head_dim);
    if (a->pairs > 0) {
        TDGS_REQUIRE(a->axes >= 1 && a->axes <= 4, "head norm: %d axes", a->axes);
        int64_t sum = 0;
        for (int i = 0; i < a->axes; ++i) {
            TDGS_REQUIRE(a->sections[i] > 0, "head norm: axis %d has %d pairs", i, a->sections[i]);
            sum += a->sections[i];
        }
        TDGS_REQUIRE(sum == a->pairs, "head norm: the axes have %lld pairs, not %d", (long long)sum, a->pairs);
        TDGS_REQUIRE(a->pair_layout == TDGS_PAIRS_HALVES || a->pair_layout == TDGS_PAIRS_INTERLEAVED,
                     "head norm: unknown layout of pairs %d", a->pair_layout);
        TDGS_REQUIRE(a->position_type >= TDGS_POSITION_I32 && a->position_type <= TDGS_POSITION_F32,
                     "head norm: unknown type of positions %d", a->position_type);
        TDGS_REQUIRE(a->turns && aligned_to(a->turns, 8), "head norm: the frequencies are null or not aligned");
        // (an empty tensor has no address)
        TDGS_REQUIRE((a->positions || a->batch == 0 || a->length == 0) &&
                         aligned_to(a->positions, a->position_type == TDGS_POSITION_I64 ? 8 : 4),
                     "head norm: the positions are null or not aligned");
        TDGS_REQUIRE(a->position_batch_stride >= 0, "head norm: positions have a negative stride");
    }
    return TDGS_OK;
}

static ByteDims hn_bytes(const tdgs_heads& v, const tdgs_head_norm* a, int heads) {
    const int64_t size = (int64_t)dtype_size(a->dtype);
    return ByteDims(v.data, {a->batch, a->length, heads}, {v.stride_b * size, v.stride_l * size, v.stride_h * size}, a->head_dim * size);
}

static int hn_check_view(const tdgs_heads* v, const char* name, const tdgs_head_norm* a, int heads, bool written) {
    TDGS_REQUIRE(v->data != nullptr, "head norm: %s is null", name);
    TDGS_REQUIRE(aligned_to(v->data, (size_t)dtype_size(a->dtype)), "head norm: %s is not aligned to its element type", name);
    TDGS_REQUIRE(v->stride_b >= 0 && v->stride_l >= 0 && v->stride_h >= 0, "head norm: %s has a negative stride", name);
    if (written)
        TDGS_REQUIRE(hn_bytes(*v, a, heads).nested, "head norm: rows of %s overlap", name);
    return TDGS_OK;
}

// A result may be what it is computed from (a head is read by the lanes that write it), and overlaps nothing else: the other result,
// what that is computed from. `read`: x, and dout or null, of queries and keys, `written` their results; null without heads.
static int hn_check_apart(const tdgs_head_norm* a, const tdgs_heads* const (&read)[2][2], const tdgs_heads* const (&written)[2],
                          const char* const (&names)[2][3]) {
    const int heads[2] = {a->heads, a->kv_heads};
    for (int i = 0; i < 2; ++i) {
        if (!written[i]) continue;
        const ByteDims w = hn_bytes(*written[i], a, heads[i]);
        for (int j = 0; j < 2; ++j) {
            for (int n = 0; n < 2; ++n) {
                if (!written[j] || !read[j][n]) continue;
                const ByteDims r = hn_bytes(*read[j][n], a, heads[j]);
                TDGS_REQUIRE(!dims_overlap(w, r) || (i == j && w.same(r)), "head norm: %s overlaps %s%s", names[i][2], names[j][n],
                             i == j ? " without being it" : "");
            }
            if (j > i && written[j])
                TDGS_REQUIRE(!dims_overlap(w, hn_bytes(*written[j], a, heads[j])), "head norm: %s overlaps %s", names[i][2], names[j][2]);
        }
    }
    return TDGS_OK;
}

struct HnPlan {
    int v, blocks;
    size_t lds;
};

// Elements a lane takes of each half: eight of a 16-bit type (16 bytes; in the gradient, whose sums for dw would then leave
// room for three wavefronts a SIMD, four: 32 heads of 64 bfloat16 146 us instead of 157) or four, where the pairs and
// what is not rotated divide into them, or single ones.
static HnPlan hn_plan(const tdgs_head_norm* a, HnArgs* r, bool grad) {
    HnPlan p;
    const int rest = a->head_dim - 2 * a->pairs;
    auto fits = [&](int v) { return a->pairs % v == 0 && rest % (2 * v) == 0; };
    p.v = a->dtype != TDGS_F32 && !grad && fits(8) ? 8 : fits(4) ? 4 : 1;
    r->rotated_units = a->pairs / p.v;
    r->units = r->rotated_units + (rest + 2 * p.v - 1) / (2 * p.v);
    r->lanes = r->units < kWave ? r->units : kWave;
    // tokens at a time: four rows per thread's lane of the fewer heads, fewer tokens where that would leave
    // compute units idle, and what LDS holds
    const int64_t tokens = (int64_t)a->batch * a->length;
    const int few = a->heads && (a->heads < a->kv_heads || !a->kv_heads) ? a->heads : a->kv_heads;
    int64_t per = ceil_div(4 * (kHnThreads / kWave) * (kWave / r->lanes), few > 0 ? few : 1);
    if (per > tokens / kHnBlocks) per = tokens / kHnBlocks;
    if (a->pairs && per > kHnAngles / a->pairs) per = kHnAngles / a->pairs;
    if (per > kHnTokens) per = kHnTokens;
    if (per < 1) per = 1;
    r->per = (int32_t)per;
    const int64_t blocks = ceil_div(tokens, per);
    const int64_t most = grad ? kHnBlocks : kHnMostBlocks;
    p.blocks = (int)(blocks < most ? blocks : most);
    p.lds = (size_t)(per * a->pairs * (int64_t)sizeof(float2));
    return p;
}

static HnArgs hn_args(const tdgs_head_norm* a) {
    HnArgs r = {};
    const tdgs_heads* const x[2] = {&a->q, &a->k};
    for (int i = 0; i < 2; ++i) {
        r.t[i].x = x[i]->data;
        r.t[i].xb = x[i]->stride_b;
        r.t[i].xl = x[i]->stride_l;
        r.t[i].xh = x[i]->stride_h;
        r.t[i].weight = i ? a->k_weight : a->q_weight;
    }
    r.turns = a->turns;
    r.positions = a->positions;
    r.position_batch = a->position_batch_stride;
    r.tokens = (int64_t)a->batch * a->length;
    r.length = a->length;
    r.heads[0] = a->heads;
    r.heads[1] = a->kv_heads;
    r.d = a->head_dim;
    r.pairs = a->pairs;
    r.axes = a->axes;
    for (int i = 0, sum = 0; i < 4; ++i) {
        if (i < a->axes && a->pairs) sum += a->sections[i];
        r.ends[i] = sum;
    }
    r.position_type = a->position_type;
    r.eps = a->eps;
    r.inv_d = 1.0f / (float)a->head_dim;
    r.sign = a->inverse ? -1.0f : 1.0f;
    r.norm = a->norm != 0;
    r.interleaved = a->pair_layout == TDGS_PAIRS_INTERLEAVED;
    r.param_f32 = a->param_dtype == TDGS_F32;
    for (int i = 0; i < 2; ++i) r.by_heads[i] = FastDiv((uint32_t)(r.heads[i] > 0 ? r.heads[i] : 1));
    r.by_pairs = FastDiv((uint32_t)(a->pairs > 0 ? a->pairs : 1));
    r.by_length = FastDiv((uint32_t)(a->length > 0 ? a->length : 1));
    return r;
}

static void hn_out(HnTensor* t, const tdgs_heads& v) {
    t->out = v.data;
    t->ob = v.stride_b;
    t->ol = v.stride_l;
    t->oh = v.stride_h;
}

// f(T{}, elements of a half per lane, units per lane, their kind)
template <class F>
static int hn_dispatch(const tdgs_head_norm* a, const HnPlan& p, F&& f) {
    using One = std::integral_constant<int, 1>;
    using Neighbours = std::integral_constant<int, kHnNeighbours>;
    const bool neighbours = a->pairs == 0 || a->pair_layout == TDGS_PAIRS_INTERLEAVED;
    return with_dtype(a->dtype, [&](auto t) -> int {
        // (single pairs: every kind is as quick as any)
        if (p.v == 1) {
            using Mixed = std::integral_constant<int, kHnMixed>;
            if (a->head_dim > 128) return neighbours ? f(t, One{}, std::integral_constant<int, 2>{}, Neighbours{})
                                                     : f(t, One{}, std::integral_constant<int, 2>{}, Mixed{});
            return neighbours ? f(t, One{}, One{}, Neighbours{}) : f(t, One{}, One{}, Mixed{});
        }
        auto kinds = [&](auto v) -> int {
            if (neighbours) return f(t, v, One{}, Neighbours{});
            if (2 * a->pairs == a->head_dim) return f(t, v, One{}, std::integral_constant<int, kHnHalves>{});
            return f(t, v, One{}, std::integral_constant<int, kHnMixed>{});
        };
        if constexpr (sizeof(t) == 2)
            if (p.v == 8) return kinds(std::integral_constant<int, 8>{});
        return kinds(std::integral_constant<int, 4>{});
    });
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

int tdgs_head_norm_forward(void* stream_, const tdgs_head_norm* a) {
    TDGS_TRY(hn_check(a));
    if (a->batch == 0 || a->length == 0 || a->heads + a->kv_heads == 0) return TDGS_OK;
    HnArgs r = hn_args(a);
    if (a->heads > 0) {
        TDGS_TRY(hn_check_view(&a->q, "q", a, a->heads, false));
        TDGS_TRY(hn_check_view(&a->q_out, "q_out", a, a->heads, true));
        hn_out(&r.t[0], a->q_out);
    }
    if (a->kv_heads > 0) {
        TDGS_TRY(hn_check_view(&a->k, "k", a, a->kv_heads, false));
        TDGS_TRY(hn_check_view(&a->k_out, "k_out", a, a->kv_heads, true));
        hn_out(&r.t[1], a->k_out);
    }
    TDGS_TRY(hn_check_apart(a, {{&a->q, nullptr}, {&a->k, nullptr}}, {a->heads > 0 ? &a->q_out : nullptr, a->kv_heads > 0 ? &a->k_out : nullptr},
                            {{"q", "", "q_out"}, {"k", "", "k_out"}}));
    const HnPlan p = hn_plan(a, &r, false);
    hipStream_t stream = (hipStream_t)stream_;
    return hn_dispatch(a, p, [&](auto t, auto v, auto n, auto kind) -> int {
        k_head_norm<decltype(t), decltype(v)::value, decltype(n)::value, decltype(kind)::value><<<(unsigned)p.blocks, kHnThreads, p.lds, stream>>>(r);
        TDGS_LAUNCHED();
        return TDGS_OK;
    });
}

size_t tdgs_head_norm_temp_bytes(const tdgs_head_norm* a) {
    if (hn_check(a) != TDGS_OK) return 0;
    const int64_t tokens = (int64_t)a->batch * a->length;   // (however the call's positions cut them)
    return align_up((size_t)(tokens < kHnBlocks ? tokens : kHnBlocks) * 2 * a->head_dim * sizeof(float));
}

int tdgs_head_norm_grad(void* stream_, const tdgs_head_norm* a, const tdgs_head_norm_grads* g) {
    TDGS_TRY(hn_check(a));
    TDGS_REQUIRE(g != nullptr, "head norm: null gradients");
    TDGS_REQUIRE(a->norm, "head norm: the gradient of a rotation alone is the inverse rotation");
    TDGS_REQUIRE(aligned_to(g->dq_weight, (size_t)dtype_size(a->param_dtype)) && aligned_to(g->dk_weight, (size_t)dtype_size(a->param_dtype)),
                 "head norm: the weights' gradients are not aligned to their element type");
    HnArgs r = hn_args(a);
    const bool empty = a->batch == 0 || a->length == 0 || a->heads + a->kv_heads == 0;
    auto view = [&](int i, const tdgs_heads& x, const tdgs_heads& d, const tdgs_heads& dx, int heads, const char* const* names) -> int {
        TDGS_TRY(hn_check_view(&x, names[0], a, heads, false));
        TDGS_TRY(hn_check_view(&d, names[1], a, heads, false));
        TDGS_TRY(hn_check_view(&dx, names[2], a, heads, true));
        r.t[i].dout = d.data;
        r.t[i].db = d.stride_b;
        r.t[i].dl = d.stride_l;
        r.t[i].dh = d.stride_h;
        hn_out(&r.t[i], dx);
        return TDGS_OK;
    };
    static const char* const kNames[2][3] = {{"q", "dq_out", "dq"}, {"k", "dk_out", "dk"}};
    if (!empty && a->heads > 0) TDGS_TRY(view(0, a->q, g->dq_out, g->dq, a->heads, kNames[0]));
    if (!empty && a->kv_heads > 0) TDGS_TRY(view(1, a->k, g->dk_out, g->dk, a->kv_heads, kNames[1]));
    HnPlan p = hn_plan(a, &r, true);
    const bool weights = g->dq_weight || g->dk_weight;
    const size_t bytes = (size_t)p.blocks * 2 * a->head_dim * sizeof(float);
    TDGS_REQUIRE(!weights || empty || (a->temp && a->temp_bytes >= bytes && aligned_to(a->temp, 16)),
                 "head norm: scratch of %zu bytes, the gradient needs %zu", a->temp ? a->temp_bytes : (size_t)0, bytes);
    if (!empty)
        TDGS_TRY(hn_check_apart(a, {{&a->q, &g->dq_out}, {&a->k, &g->dk_out}},
                                {a->heads > 0 ? &g->dq : nullptr, a->kv_heads > 0 ? &g->dk : nullptr}, kNames));
    hipStream_t stream = (hipStream_t)stream_;
    r.part = weights ? (float*)a->temp : nullptr;
    if (empty) p.blocks = 0;   // (the weights' gradients are zero)
    return hn_dispatch(a, p, [&](auto t, auto v, auto n, auto kind) -> int {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        if constexpr (V <= 4) {
            if (!empty) {
                k_head_norm_grad<T, V, decltype(n)::value, decltype(kind)::value><<<(unsigned)p.blocks, kHnThreads, p.lds, stream>>>(r);
                TDGS_LAUNCHED();
            }
        }
        if (weights) {
            k_head_norm_join<T><<<(unsigned)ceil_div(2 * a->head_dim, kHnJoinCols), kHnThreads, 0, stream>>>(
                r.part, p.blocks, a->head_dim, g->dq_weight, g->dk_weight, r.param_f32);
            TDGS_LAUNCHED();
        }
        return TDGS_OK;
    });
}

}  // extern "C"
