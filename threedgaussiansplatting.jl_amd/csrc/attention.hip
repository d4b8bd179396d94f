// attention.hip — cross attention of a decoder's queries to an encoder's states, forward and
// backward, on the matrix cores.
//
// The query heads that share a kv head, and the query batches that share an encoder's states, are
// stacked into the rows of one problem per kv head and kv batch: row r is query
// (r / (q_len G)) of the sharing batches, r / G % q_len of its queries and r % G of the G heads. A tile
// of keys is so staged once for all of them, and a single query token of G heads fills G rows.
//
// Products are 32x32 blocks (elem.hpp). Scores are taken as S^T = K Q^T in the forward pass and for
// dQ: a lane then holds 16 keys of one row, the softmax's maximum and sum are in-lane but for one
// swap of the halves, and P^T is in place as the next product's B operand (O^T = V^T P^T,
// dQ^T = K^T dS^T), V^T and K^T coming from LDS by the transposing reads. For dK and dV the block is
// S = Q K^T, a lane holding 16 rows of one key, and dV^T = dO^T P, dK^T = Q^T dS follow likewise.
// A key mask is turned into a list of the allowed keys first, by which keys are then loaded and their
// gradients stored, so that the kernels see a shorter sequence: they do no work for single keys that are not allowed,
// and such keys, whatever they hold, are not read.
// P and dS are rounded to the inputs' type for their products (the matrix cores take no wider
// operand at that rate), in half after a power of two that brings them into its range; maxima, sums,
// exponentials and every accumulator stay in 32 bits.
//
// What bounds the kernels: for 16-bit types the exponential of every score, at a quarter of the vector rate, next to
// the products; for float the products themselves; for few rows over many keys the memory that
// the keys are read from; for few rows and keys the latency of one or two tiles. Measured figures stand at each kernel.
#include "internal.hpp"
#include "elem.hpp"

namespace tdgs {

constexpr int kAtThreads = 256;
constexpr int kAtWaves = kAtThreads / kWave;
constexpr float kLn2 = 0.69314718055994530942f;

struct AtHeads {
    int64_t b, l, h;   // strides in elements
};

struct AtArgs {
    const void *q, *k, *v, *dout, *o;
    void *out, *dq, *dk, *dv;
    AtHeads sq, sk, sv, so, sdo, sdq, sdk, sdv;
    const int32_t* lengths;   // allowed keys of a kv batch (with a mask: of its list); null: all
    const int32_t* index;     // with a mask: kv_len keys of each kv batch, the allowed ones first
    float* lse;       // batch x heads x q_len, natural logarithm
    float* delta;     // the same shape: dout . out
    float *part, *part_ml;
    int32_t q_len, kv_len, heads, kv_heads, d;
    int32_t rows;     // per kv head and kv batch
    int32_t group_batches, splits, blocks;
    float c, scale;   // scale log2(e), scale
    FastDiv by_g, by_lg;
    bool vec_out;
};

struct AtRow {
    int32_t b, i, h;   // batch, query, head
};

__device__ __forceinline__ AtRow at_row(const AtArgs& a, int kb, int hk, int r) {
    const uint32_t bb = a.by_lg.div(r), rest = r - bb * a.by_lg.d, i = a.by_g.div(rest);
    return {kb * a.group_batches + (int32_t)bb, (int32_t)i, hk * (int32_t)a.by_g.d + (int32_t)(rest - i * a.by_g.d)};
}
__device__ __forceinline__ int64_t at_offset(const AtHeads& s, const AtRow& r) {
    return r.b * s.b + r.i * s.l + r.h * s.h;
}
__device__ __forceinline__ int64_t at_stat(const AtArgs& a, const AtRow& r) {
    return ((int64_t)r.b * a.heads + r.h) * a.q_len + r.i;
}

__device__ __forceinline__ int at_length(const AtArgs& a, int kb) {
    if (!a.lengths) return a.kv_len;
    const int n = a.lengths[kb];
    return n < 0 ? 0 : (n < a.kv_len ? n : a.kv_len);
}

__device__ __forceinline__ int64_t at_key(const AtArgs& a, int kb, int j) {
    return a.index ? a.index[(int64_t)kb * a.kv_len + j] : j;
}

// Workgroup kb: the list of kv batch kb's keys, the allowed ones first and in order, and their number.
constexpr int kAtListThreads = 1024;
static __global__ __launch_bounds__(kAtListThreads) void k_attend_list(const uint8_t* __restrict__ mask, int64_t stride,
                                                                       AtArgs a, int32_t* __restrict__ index,
                                                                       int32_t* __restrict__ counts) {
    constexpr int PER = 4, W = kAtListThreads / kWave;
    __shared__ int s_wave[W];
    const int kb = blockIdx.x, lane = (int)__lane_id(), wave = threadIdx.x / kWave, len = at_length(a, kb);
    const uint8_t* const row = mask + kb * stride;
    int32_t* const list = index + (int64_t)kb * a.kv_len;
    int done = 0;   // allowed keys before these
    for (int r0 = 0; r0 < a.kv_len; r0 += kAtListThreads * PER) {
        // a wavefront takes PER * 64 neighbouring keys
        const int j0 = r0 + wave * (kWave * PER) + lane;
        uint64_t votes[PER];
        bool ok[PER];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = j0 + i * kWave;
            ok[i] = j < len && row[j] != 0;
            votes[i] = __ballot(ok[i]);
            mine += __popcll(votes[i]);
        }
        if (lane == 0) s_wave[wave] = mine;
        __syncthreads();
        int at = done;
        for (int w = 0; w < W; ++w) {
            const int c = s_wave[w];
            if (w < wave) at += c;
            done += c;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = j0 + i * kWave, before = at + __popcll(votes[i] & lanemask_lt());
            if (j < a.kv_len) list[ok[i] ? before : a.kv_len - 1 - (j - before)] = j;   // (the others from the end on)
            at += __popcll(votes[i]);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) counts[kb] = done;
}

// Keys per tile of the forward and dQ kernels, and rows per tile of the dK, dV kernel. LDS rows are
// padded by 16 bytes: for every DP, a b128 read of one depth chunk of 16 rows then covers the 64
// banks exactly once.
template <class T>
constexpr int at_tile() { return sizeof(T) == 4 ? 32 : 64; }
template <class T, int DP>
constexpr int at_pitch() { return DP + 16 / (int)sizeof(T); }

// One tile of N rows x DP elements in registers on its way to LDS, thread t of TH taking chunks of eight
// elements t, t + TH, .. VEC: rows start on 16 bytes and d is a multiple of 8. Such chunks are loaded
// without a condition, from an element that exists, and replaced by zeros on their way to LDS where they
// should not count: a load behind a branch is waited for at its end, not where it is used.
template <class T, int DP, int N, int TH, bool VEC>
struct AtTile {
    static constexpr int kChunks = N * (DP / 8);
    static constexpr int kPer = (kChunks + TH - 1) / TH;
    typename Elem<T>::V8 r[kPer];
    __device__ __forceinline__ static int chunk(int k) { return (int)threadIdx.x + k * TH; }
    __device__ __forceinline__ static bool inside(int k) { return kChunks % TH == 0 || chunk(k) < kChunks; }
    __device__ __forceinline__ static int row(int k) { return chunk(k) / (DP / 8); }
    __device__ __forceinline__ static int col(int k) { return chunk(k) % (DP / 8) * 8; }
    // Chunk k from the row at p (any readable row for one that does not count).
    __device__ __forceinline__ void load_row(int k, const T* p, int d) {
        if constexpr (VEC) r[k] = *reinterpret_cast<const typename Elem<T>::V8a*>(p + (col(k) < d ? col(k) : 0));
        else r[k] = load8<T>(p + col(k), d - col(k), false);
    }
    // Rows first.. of those at base + j * stride (j from `index` where not null, with IDX), of which `rows` > 0 are
    // left. Only the addresses are made behind branches.
    template <bool IDX>
    __device__ __forceinline__ void load(const T* base, int64_t stride, const int32_t* index, int first, int rows, int d) {
        const T* p[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) p[k] = base + first * stride + min(inside(k) ? row(k) : 0, rows - 1) * stride;
        if (IDX && index) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) p[k] = base + index[first + min(inside(k) ? row(k) : 0, rows - 1)] * stride;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) load_row(k, p[k], d);
    }
    // To LDS; then zeros over what lies past the `rows` that are left, or past d.
    __device__ __forceinline__ void store(T* lds, int rows, int d) const {
        auto at = [&](int k) {
            return reinterpret_cast<typename Elem<T>::V8a*>(lds + row(k) * at_pitch<T, DP>() + col(k));
        };
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (inside(k)) *at(k) = r[k];
        if (rows < N || d < DP) {
#pragma unroll
            for (int k = 0; k < kPer; ++k)
                if (inside(k) && (row(k) >= rows || col(k) >= d)) *at(k) = zero8<T>();
        }
    }
};

// A operand: rows base.. of the tile, depth chunk c (slot (l / 32) * 8 + i is element 16 c + that).
template <class T, int DP>
__device__ __forceinline__ typename Elem<T>::V8 at_rows(const T* lds, int base, int c) {
    const int l = (int)__lane_id();
    return *reinterpret_cast<const typename Elem<T>::V8a*>(lds + (base + (l & 31)) * at_pitch<T, DP>() + c * 16 +
                                                           (l >> 5) * 8);
}
// A operand of the transposed tile: its rows are the tile's columns db * 32.., its depth the 16 tile
// rows from base on, in the order the registers of a block of results hold them: slot (h, i) is row
// base + (i / 4) * 8 + h * 4 + i % 4. For 16-bit types two transposing reads: 16 lanes give the
// addresses of 4 rows x 16 columns and each gets one column.
template <class T, int DP>
__device__ __forceinline__ typename Elem<T>::V8 at_cols(const T* lds, int base, int db) {
    const int l = (int)__lane_id();
    typename Elem<T>::V8 r;
    if constexpr (sizeof(T) == 4) {
        const T* p = lds + (base + (l >> 5) * 4) * at_pitch<T, DP>() + db * 32 + (l & 31);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = p[((i >> 2) * 8 + (i & 3)) * at_pitch<T, DP>()];
    } else {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        const T* p = lds + (base + (l >> 5) * 4 + ((l & 15) >> 2)) * at_pitch<T, DP>() + db * 32 + ((l >> 4) & 1) * 16 +
                     (l & 3) * 4;
        typedef __attribute__((address_space(3))) s4* lp;
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 8 * at_pitch<T, DP>()));
        r = __builtin_bit_cast(typename Elem<T>::V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return r;
}

// Eight registers of a block of results as an operand, rounded to T.
template <class T>
__device__ __forceinline__ typename Elem<T>::V8 at_pack(const f32x16& s, int half) {
    typename Elem<T>::V8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)s[half * 8 + i];
    return r;
}

// The same as a sum of two operands of a 16-bit type: what the rounding to T leaves goes into `rest`.
template <class T>
__device__ __forceinline__ void at_pack2(const f32x16& s, int half, typename Elem<T>::V8& r, typename Elem<T>::V8& rest) {
    if constexpr (std::is_same<T, bf16>::value) {   // (the upper halves as they are: what they leave is exact either way)
        uint32_t hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float fx = s[half * 8 + 2 * i], fy = s[half * 8 + 2 * i + 1];   // (copies: this compiler casts element 0
            const uint32_t x = __builtin_bit_cast(uint32_t, fx), y = __builtin_bit_cast(uint32_t, fy);   // of a vector only)
            hi[i] = __builtin_amdgcn_perm(y, x, 0x07060302);
            rest[2 * i] = (T)(fx - __builtin_bit_cast(float, x & 0xffff0000u));
            rest[2 * i + 1] = (T)(fy - __builtin_bit_cast(float, y & 0xffff0000u));
        }
        typedef uint32_t U4 __attribute__((ext_vector_type(4)));
        const U4 v = {hi[0], hi[1], hi[2], hi[3]};
        r = __builtin_bit_cast(typename Elem<T>::V8, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            r[i] = (T)s[half * 8 + i];
            rest[i] = (T)(s[half * 8 + i] - (float)r[i]);
        }
    }
}

// Eight registers of a block of results S as an operand: acc + A S. Rounded to T, or with TWO as two operands of a 16-bit
// type, by which S keeps 16 or more bits at the price of a second product.
template <class T, bool TWO>
struct AtOperand {
    static constexpr bool kTwo = TWO && sizeof(T) == 2;
    typename Elem<T>::V8 b, rest;
    __device__ __forceinline__ AtOperand(const f32x16& s, int half) {
        if constexpr (kTwo) at_pack2<T>(s, half, b, rest);
        else b = at_pack<T>(s, half);
    }
    __device__ __forceinline__ f32x16 product(typename Elem<T>::V8 a, f32x16 acc) const {
        if constexpr (kTwo) acc = mma(a, rest, acc);
        return mma(a, b, acc);
    }
};

// Brings dS into the range of its operand. A lane's registers hold dS of one row (dQ) or one key (dK), whose result no
// other lane but its partner in the other half of the wavefront adds to, so each takes its own power of two out of it.
// bfloat16 and float hold any dS; half would make infinities of those above 65504, which a scaled loss reaches, and lose
// bits of those below 6e-5, which a mean over many pixels gives. g, by which dS is multiplied, starts above all that half's
// q, k, v and dout can make (|dP| is at least 2^-48 or 0, and 2^40 at most) and is lowered, with what was added up before,
// where dS would pass 2^15; the largest dS is then brought to 2^8, so that it may grow 2^7 times before that happens
// again. Forward and backward of 64800 rows x 1024 keys x 8 heads of 64 take 833 us with it, 804 without.
template <class T>
struct AtRange {
    static constexpr bool kOn = std::is_same<T, f16>::value;
    float g = kOn ? 0x1p64f : 1.0f;
    // Whether x, which is g dS, is out of range; then by what it and everything added up has to be multiplied, in *f.
    __device__ __forceinline__ bool lower(const f32x16& x, float* f) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
        if (!wave_any(top > 0x1p15f)) return false;
        top = max_halves(top);
        *f = 1.0f;
        if (top > 0x1p15f) {   // (infinity: 2^-120)
            *f = __builtin_bit_cast(float, (uint32_t)((8 + 2 * 127) << 23) - (__builtin_bit_cast(uint32_t, top) & 0x7f800000u));
            g *= *f;
        }
        return true;
    }
    __device__ __forceinline__ float undo() const {   // 1 / g
        return kOn ? __builtin_bit_cast(float, (uint32_t)(2 * 127 << 23) - __builtin_bit_cast(uint32_t, g)) : 1.0f;
    }
};

// P is at most 1 in the backward pass, and over many keys small: half takes 2^14 P.
template <class T>
constexpr float at_p_shift() { return std::is_same<T, f16>::value ? 14.0f : 0.0f; }
template <class T>
constexpr float at_p_undo() { return std::is_same<T, f16>::value ? 0x1p-14f : 1.0f; }

// Row r's elements in the order of a B operand's lanes (row l % 32 of the block): chunk c of DP / 16.
template <class T, int DP, bool VEC>
__device__ __forceinline__ void at_load_row(typename Elem<T>::V8 (&f)[DP / 16], const T* p, int d) {
    const int h = (int)__lane_id() >> 5;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        const int e = c * 16 + h * 8;
        if constexpr (VEC) {
            if (p && e < d) f[c] = *reinterpret_cast<const typename Elem<T>::V8a*>(p + e);
            else f[c] = zero8<T>();
        } else {
            f[c] = p ? load8<T>(p + e, d - e, false) : zero8<T>();
        }
    }
}

template <class V2>
__device__ __forceinline__ uint32_t at_bits(V2 v) {
    return __builtin_bit_cast(uint32_t, v);
}

template <class T>
__device__ __forceinline__ void at_store4(T* p, f32x4 x, int n, bool vec) {
    if (vec && n >= 4) {
        typedef T V4a __attribute__((ext_vector_type(4), aligned(8)));
        V4a r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (T)x[i];
        *reinterpret_cast<V4a*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = (T)x[i];
    }
}

// A block column of results (d x 32 lanes' rows, DP / 32 blocks) times f to a row of T. A lane holds four
// elements in eight, its partner in the other half of the wavefront the other four: rows of a 16-bit type that
// allow it trade two fours of theirs for one eight, and store 16 bytes (every lane of the
// wavefront calls this; p null: nothing stored).
template <class T, int DP>
__device__ __forceinline__ void at_store_row(T* p, const f32x16 (&o)[DP / 32], float f, int d, bool vec) {
    const int h = (int)__lane_id() >> 5;
    if constexpr (sizeof(T) == 2) if (vec) {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                uint32_t x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    typedef T V2 __attribute__((ext_vector_type(2)));
                    const V2 lo = {(T)(o[db][k * 4 + 2 * i] * f), (T)(o[db][k * 4 + 2 * i + 1] * f)};
                    const V2 hi = {(T)(o[db][k * 4 + 4 + 2 * i] * f), (T)(o[db][k * 4 + 5 + 2 * i] * f)};
                    const auto r = __builtin_amdgcn_permlane32_swap(at_bits(lo), at_bits(hi), false, false);
                    x[i] = r[0];
                    y[i] = r[1];
                }
                const int e = db * 32 + (k + h) * 8;
                typedef uint32_t U4 __attribute__((ext_vector_type(4)));
                const U4 v = {x[0], x[1], y[0], y[1]};
                if (p && e < d) *reinterpret_cast<U4*>(p + e) = v;
            }
        return;
    }
    if (!p) return;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = db * 32 + k * 8 + h * 4;
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = o[db][k * 4 + i] * f;
            at_store4<T>(p + e, x, d - e, vec);
        }
}

// Kernels that share rows' heads: the workgroup of (kv head, rest), heads next to each other on one XCD. Neighbouring
// heads of a row share its cache lines, so their workgroups should share an L2 (workgroup i runs on XCD
// i mod 8). Keys of a head are read by many workgroups, but a band of them for each XCD gains 1 to 2% where every
// head has much to do (32400 x 4096) and loses as much where not, and where lengths or masks differ between
// batches leaves whole XCDs without work.
struct AtItem {
    int hk, rest;
};
__device__ __forceinline__ AtItem at_item(int i, int n, int kv_heads) {
    const int whole = n / (kXcds * kv_heads) * (kXcds * kv_heads);
    if (i >= whole) return {i % kv_heads, i / kv_heads};
    const int j = i / kXcds;
    return {j % kv_heads, j / kv_heads * kXcds + i % kXcds};
}

// How far below the largest c s of a tile its row's reference m is put, and what a lane's p of a tile may add up to
// before m is looked for again: 2^10 times that of the largest. In half both are up by 2^5, and p stays below 2^15: weights
// down to 2^-19 of the largest so keep all of half's bits, which matters where the key that has it has no value.
template <class T>
constexpr float at_below() { return std::is_same<T, f16>::value ? 5.0f : 0.0f; }
template <class T>
constexpr float at_largest() { return std::is_same<T, f16>::value ? 0x1p15f : 0x1p10f; }
constexpr float kAtLowest = -1e38f;   // below any score: what m starts from

// The forward kernel's workgroup: threads, and wavefronts per SIMD that its registers leave room for. With 512
// threads and four per SIMD a tile is staged once for 256 rows and the wavefronts cover each other's waits; two
// blocks of rows per wavefront, or one wavefront per SIMD with twice the registers, were 0 to 70% slower.
template <class T, int DP>
struct AtForward {
    static constexpr int kThreads = sizeof(T) == 2 && DP <= 64 ? 512 : 256;
    static constexpr int kPerSimd = sizeof(T) == 2 && DP <= 64 ? 4 : 2;
    static constexpr int kRows = kThreads / kWave * 32;
};

// Workgroup: wavefronts of 32 rows each of one kv head, the keys of one split. Softmax in base 2: O and l are
// relative to m, the largest c s of the first tile. It need not be the largest so far: only when a later tile's
// p add up to more than at_largest are the scores taken again, m moved to their largest and O and l brought there, so
// that almost every tile does without finding a maximum (5% of the kernel).
// bfloat16, heads of 64: 64800 rows x 1024 keys x 8 heads in 162 to 184 us (136 GFLOP: 740 to 840 TFLOP/s; a large
// product reaches 1150), vector issue busy for 64% of it, the matrix cores for 38%; 32400 x 4096 x 16 in 594 us when
// the card is cool, 760 when not (910 to 710 TFLOP/s at 2.1 to 1.7 GHz). float: matrix cores busy for half of the time.
// One row of 16 heads over 8 caches of 10000 to 20011 keys: 40 us, 6 TB/s.
template <class T, int DP, bool VEC, bool IDX, bool TWO>
__global__ __launch_bounds__((AtForward<T, DP>::kThreads), (AtForward<T, DP>::kPerSimd)) void k_attend(AtArgs a) {
    constexpr int TH = AtForward<T, DP>::kThreads;
    constexpr int KT = at_tile<T>(), P = at_pitch<T, DP>(), NB = DP / 32, NC = DP / 16, NK = KT / 32;
    __shared__ __attribute__((aligned(16))) T s_k[KT * P];
    __shared__ __attribute__((aligned(16))) T s_v[KT * P];
    const AtItem item = at_item(blockIdx.x, gridDim.x, a.kv_heads);
    const int blk = item.rest % a.blocks, sp = item.rest / a.blocks % a.splits, kb = item.rest / a.blocks / a.splits;
    const int hk = item.hk, kvh = kb * a.kv_heads + hk;
    const int lane = (int)__lane_id(), wave = threadIdx.x / kWave, h = lane >> 5;
    const int r = blk * AtForward<T, DP>::kRows + wave * 32 + (lane & 31);
    const bool in = r < a.rows;

    typename Elem<T>::V8 qf[NC];
    at_load_row<T, DP, VEC>(qf, in ? (const T*)a.q + at_offset(a.sq, at_row(a, kb, hk, r)) : nullptr, a.d);
    f32x16 o[NB];
    float m = kAtLowest, l = 0.0f;
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    const bool busy = blk * AtForward<T, DP>::kRows + wave * 32 < a.rows;   // (the others only bring keys)
    const int len = at_length(a, kb);
    const int tiles = (len + KT - 1) / KT, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = sp * per, t_end = min(tiles, t0 + per);
    const T* const kbase = (const T*)a.k + kb * a.sk.b + hk * a.sk.h;
    const T* const vbase = (const T*)a.v + kb * a.sv.b + hk * a.sv.h;
    AtTile<T, DP, KT, TH, VEC> tk, tv;
    const int32_t* const index = IDX && a.index ? a.index + (int64_t)kb * a.kv_len : nullptr;
    auto fetch = [&](int t) {
        tk.template load<IDX>(kbase, a.sk.l, index, t * KT, len - t * KT, a.d);
        tv.template load<IDX>(vbase, a.sv.l, index, t * KT, len - t * KT, a.d);
    };
    f32x16 s[NK];
    auto scores = [&](int left) {
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kk][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c) s[kk] = mma(at_rows<T, DP>(s_k, kk * 32, c), qf[c], s[kk]);
        }
        if (left < KT) {
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[kk][i] = kk * 32 + (i >> 2) * 8 + (i & 3) < left - h * 4 ? s[kk][i] : -INFINITY;
        }
    };
    auto move = [&]() {   // m to the largest score so far
        float top = s[0][0];
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kk][i]);
        top = fmaxf(max_halves(top) * a.c - at_below<T>(), m);
        const float f = __builtin_amdgcn_exp2f(m - top);
        l *= f;
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= f;
        m = top;
    };
    auto weights = [&]() {   // p in place of the scores; their sum
        float sum = 0.0f;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kk][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk][i], a.c, -m));
                sum += s[kk][i];
            }
        return sum;
    };
    if (t0 < t_end) fetch(t0);
    for (int t = t0; t < t_end; ++t) {
        const int left = len - t * KT;
        __syncthreads();
        tk.store(s_k, left, a.d);
        tv.store(s_v, left, a.d);
        __syncthreads();
        if (t + 1 < t_end) fetch(t + 1);
        if (!busy) continue;
        scores(left);
        if (t == t0) move();
        float sum = weights();
        if (wave_any(!(sum <= at_largest<T>()))) {   // (NaN too, and then stays)
            scores(left);
            move();
            sum = weights();
        }
        l += sum;
#pragma unroll
        for (int ks = 0; ks < KT / 16; ++ks) {
            const AtOperand<T, TWO> p(s[ks / 2], ks % 2);
#pragma unroll
            for (int db = 0; db < NB; ++db) o[db] = p.product(at_cols<T, DP>(s_v, ks * 16, db), o[db]);
        }
    }
    l = sum_halves(l);
    if (a.splits == 1) {
        const AtRow row = at_row(a, kb, hk, in ? r : 0);
        at_store_row<T, DP>(in ? (T*)a.out + at_offset(a.so, row) : nullptr, o, l > 0.0f ? 1.0f / l : 0.0f, a.d, a.vec_out);
        if (in && a.lse && h == 0) a.lse[at_stat(a, row)] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    } else if (in) {
        const int64_t pr = ((int64_t)sp * gridDim.x / (a.blocks * a.splits) + kvh) * a.rows + r;
        at_store_row<float, DP>(a.part + pr * DP, o, 1.0f, DP, true);
        if (h == 0) {
            a.part_ml[2 * pr] = m;
            a.part_ml[2 * pr + 1] = l;
        }
    }
}

// Joins the splits of a row: O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s. A thread holds four
// elements of a row; with SG > 1, for many splits of few rows, SG of them take every SG-th split and
// are joined likewise in LDS. 128 rows of 32 splits: 4.6 us, nearly all latency; 60024 float rows of 64 elements
// in two splits: 11 us, 4.1 TB/s.
template <class T, int SG>
__global__ __launch_bounds__(kAtThreads) void k_attend_join(AtArgs a, int dp, int64_t all_rows) {
    __shared__ f32x4 s_x[SG > 1 ? kAtThreads : 1];
    __shared__ float2 s_ml[SG > 1 ? kAtThreads : 1];
    const int quads = dp / 4, q = (int)threadIdx.x % quads, slot = (int)threadIdx.x / quads;
    const int per = kAtThreads / quads / SG, g = slot / per;   // rows per workgroup; this thread's share of the splits
    const int64_t pr0 = (int64_t)blockIdx.x * per + slot % per;
    const bool in = g < SG && pr0 < all_rows;
    float top = kAtLowest, sum = 0.0f;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in) {
        const float2* const ml = reinterpret_cast<const float2*>(a.part_ml) + pr0;
#pragma unroll 8
        for (int s = g; s < a.splits; s += SG) top = fmaxf(top, ml[s * all_rows].x);
        const f32x4* const part = reinterpret_cast<const f32x4*>(a.part + pr0 * dp) + q;
#pragma unroll 4
        for (int s = g; s < a.splits; s += SG) {
            const float2 v = ml[s * all_rows];
            const float f = __builtin_amdgcn_exp2f(v.x - top);
            x += *(part + s * all_rows * quads) * f;
            sum = __builtin_fmaf(f, v.y, sum);
        }
    }
    if constexpr (SG > 1) {
        s_x[threadIdx.x] = x;
        s_ml[threadIdx.x] = make_float2(top, sum);
        __syncthreads();
        if (g == 0) {
            const int step = per * quads;
            for (int i = 1; i < SG; ++i) top = fmaxf(top, s_ml[threadIdx.x + i * step].x);
            x = {0.0f, 0.0f, 0.0f, 0.0f};
            sum = 0.0f;
            for (int i = 0; i < SG; ++i) {
                const float2 v = s_ml[threadIdx.x + i * step];
                const float f = __builtin_amdgcn_exp2f(v.x - top);
                x += s_x[threadIdx.x + i * step] * f;
                sum = __builtin_fmaf(f, v.y, sum);
            }
        }
    }
    if (!in || g > 0) return;
    const int kvh = (int)(pr0 / a.rows);
    const AtRow row = at_row(a, kvh / a.kv_heads, kvh % a.kv_heads, (int)(pr0 % a.rows));
    if (q * 4 < a.d)
        at_store4<T>((T*)a.out + at_offset(a.so, row) + q * 4, x * (sum > 0.0f ? 1.0f / sum : 0.0f), a.d - q * 4, a.vec_out);
    if (a.lse && q == 0) a.lse[at_stat(a, row)] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ---- backward ------------------------------------------------------------------------------

// The base-2 logarithm of a row's sum, from lse; +inf (all its p are 0) for a row without allowed keys.
__device__ __forceinline__ float at_lse2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// The factor of dQ and dK. The softmax of a single key is constant: its dP - delta is nothing but rounding.
__device__ __forceinline__ float at_grad_scale(const AtArgs& a, int len) { return len > 1 ? a.scale : 0.0f; }

// dQ and delta. Workgroup: 4 wavefronts of 32 rows each, the keys of one split. 16-bit types up to 64 elements take three
// per SIMD: 512 threads, two blocks of rows per wavefront, or tiles in two or three buffers were slower. Bound by vector
// issue (72% busy, the matrix cores 44%): 64800 rows x 1024 keys x 8 heads of 64, bfloat16, in 296 to 329 us (204 GFLOP of
// the formulas, 272 with the second product of dS: 830 to 920 TFLOP/s).
template <class T, int DP, bool VEC, bool IDX>
__global__ __launch_bounds__(kAtThreads, (sizeof(T) == 2 && DP <= 64 ? 3 : 2)) void k_attend_dq(AtArgs a) {
    constexpr int KT = at_tile<T>(), P = at_pitch<T, DP>(), NB = DP / 32, NC = DP / 16;
    __shared__ __attribute__((aligned(16))) T s_k[KT * P];
    __shared__ __attribute__((aligned(16))) T s_v[KT * P];
    const AtItem item = at_item(blockIdx.x, gridDim.x, a.kv_heads);
    const int blk = item.rest % a.blocks, sp = item.rest / a.blocks % a.splits, kb = item.rest / a.blocks / a.splits;
    const int hk = item.hk, kvh = kb * a.kv_heads + hk;
    const int lane = (int)__lane_id(), wave = threadIdx.x / kWave, h = lane >> 5;
    const int r = (blk * kAtWaves + wave) * 32 + (lane & 31);
    AtRow row = {0, 0, 0};
    if (r < a.rows) row = at_row(a, kb, hk, r);

    typename Elem<T>::V8 qf[NC], df[NC];
    at_load_row<T, DP, VEC>(qf, r < a.rows ? (const T*)a.q + at_offset(a.sq, row) : nullptr, a.d);
    at_load_row<T, DP, VEC>(df, r < a.rows ? (const T*)a.dout + at_offset(a.sdo, row) : nullptr, a.d);
    float lse2 = INFINITY, delta = 0.0f;
    {
        typename Elem<T>::V8 of[NC];
        at_load_row<T, DP, VEC>(of, r < a.rows ? (const T*)a.o + at_offset(a.so, row) : nullptr, a.d);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) delta = __builtin_fmaf((float)df[c][i], (float)of[c][i], delta);
        delta = sum_halves(delta);
        if (r < a.rows) lse2 = at_lse2(a.lse[at_stat(a, row)]);
    }
    f32x16 o[NB];
    AtRange<T> range;
    float lse2g = lse2 - (AtRange<T>::kOn ? 64.0f : 0.0f);   // P comes out multiplied by g
    float slip = 0.0f;   // the row's sum of dS (times g), which an exact delta makes zero
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    const bool busy = (blk * kAtWaves + wave) * 32 < a.rows;
    const int len = at_length(a, kb);
    const int tiles = (len + KT - 1) / KT, per = (tiles + a.splits - 1) / a.splits;
    const int t_end = min(tiles, (sp + 1) * per);
    const T* const kbase = (const T*)a.k + kb * a.sk.b + hk * a.sk.h;
    const T* const vbase = (const T*)a.v + kb * a.sv.b + hk * a.sv.h;
    AtTile<T, DP, KT, kAtThreads, VEC> tk, tv;
    const int32_t* const index = IDX && a.index ? a.index + (int64_t)kb * a.kv_len : nullptr;
    auto fetch = [&](int t) {
        tk.template load<IDX>(kbase, a.sk.l, index, t * KT, len - t * KT, a.d);
        tv.template load<IDX>(vbase, a.sv.l, index, t * KT, len - t * KT, a.d);
    };
    if (sp * per < t_end) fetch(sp * per);
    for (int t = sp * per; t < t_end; ++t) {
        const int left = len - t * KT;
        __syncthreads();
        tk.store(s_k, left, a.d);
        tv.store(s_v, left, a.d);
        __syncthreads();
        if (t + 1 < t_end) fetch(t + 1);
        if (!busy) continue;
        if (sizeof(T) == 2 && len <= KT) {
            // the row's sum of p dp instead of dout . out, whose rounding would show where few keys share a row
            delta = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KT / 32; ++kk) {
                f32x16 s, dp;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    s = mma(at_rows<T, DP>(s_k, kk * 32, c), qf[c], s);
                    dp = mma(at_rows<T, DP>(s_v, kk * 32, c), df[c], dp);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = kk * 32 + (i >> 2) * 8 + (i & 3) < left - h * 4 ? s[i] : -INFINITY;
                    delta = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x, a.c, -lse2)), dp[i], delta);
                }
            }
            delta = sum_halves(delta);
        }
#pragma unroll
        for (int kk = 0; kk < KT / 32; ++kk) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = mma(at_rows<T, DP>(s_k, kk * 32, c), qf[c], s);
                dp = mma(at_rows<T, DP>(s_v, kk * 32, c), df[c], dp);
            }
            if (left < KT) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[i] = kk * 32 + (i >> 2) * 8 + (i & 3) < left - h * 4 ? s[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -lse2g)) * (dp[i] - delta);
                slip += s[i];
            }
            if constexpr (AtRange<T>::kOn) {
                float f;
                if (range.lower(s, &f)) {
                    s *= f;
                    slip *= f;
                    lse2g -= __builtin_amdgcn_logf(f);
#pragma unroll
                    for (int db = 0; db < NB; ++db) o[db] *= f;
                }
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const AtOperand<T, true> b(s, ks);
#pragma unroll
                for (int db = 0; db < NB; ++db) o[db] = b.product(at_cols<T, DP>(s_k, kk * 32 + ks * 16, db), o[db]);
            }
        }
    }
    // dK takes delta with what the rows' sums have shown to be its error; over several splits the join adds it up
    slip = sum_halves(slip) * range.undo();
    if (h == 0 && r < a.rows) {
        if (a.splits == 1) a.delta[at_stat(a, row)] = delta + slip;
        else a.part_ml[((int64_t)sp * gridDim.x / (a.blocks * a.splits) + kvh) * a.rows + r] = sp == 0 ? delta + slip : slip;
    }
    if (a.splits == 1) {
        at_store_row<T, DP>(r < a.rows ? (T*)a.dq + at_offset(a.sdq, row) : nullptr, o, at_grad_scale(a, len) * range.undo(),
                            a.d, a.vec_out);
    } else if (r < a.rows) {
        const int64_t pr = ((int64_t)sp * gridDim.x / (a.blocks * a.splits) + kvh) * a.rows + r;
        at_store_row<float, DP>(a.part + pr * DP, o, range.undo(), DP, true);
    }
}

// Two wavefronts per SIMD, though heads of 97 to 128 elements then keep some registers in memory: without,
// and one wavefront, 16-bit types take 1145 us for 64800 rows, 1024 keys and 8 heads where two take 1061.
// Only float's 187 registers cost more than the second wavefront gives (5548 us, 4477 with one).
template <class T, int DP>
constexpr int at_dkv_per_simd() { return sizeof(T) == 4 && DP > 96 ? 1 : 2; }

// dK and dV. Workgroup: TH / 64 wavefronts of 32 keys each, the rows of one split. Wide ones, of 256 keys, stage rows half as
// often and 64 at a time: 343 -> 311 us for 64800 rows, 1024 keys and 8 heads of bfloat16; with 93 keys half
// their wavefronts idle (30 -> 37). The matrix cores are busy for 44% of that, LDS for 48%, vector issue for 40%
// (272 GFLOP: 860 to 980 TFLOP/s), and wavefronts wait for 36%: no unit bounds it; for float the matrix cores for 51%.
constexpr int kAtWide = 512;
template <class T, int DP, int TH, bool VEC, bool TWO>
__global__ __launch_bounds__(TH, (at_dkv_per_simd<T, DP>())) void k_attend_dkv(AtArgs a) {
    constexpr int RT = TH == kAtWide ? 64 : 32, P = at_pitch<T, DP>(), NB = DP / 32, NC = DP / 16;
    __shared__ __attribute__((aligned(16))) T s_q[RT * P];
    __shared__ __attribute__((aligned(16))) T s_d[RT * P];
    __shared__ __attribute__((aligned(16))) float s_lse[RT];
    __shared__ __attribute__((aligned(16))) float s_delta[RT];
    const int item = blockIdx.x;
    const int sp = item % a.splits, blk = item / a.splits % a.blocks, kvh = item / a.splits / a.blocks;
    const int hk = kvh % a.kv_heads, kb = kvh / a.kv_heads;
    const int lane = (int)__lane_id(), wave = threadIdx.x / kWave, h = lane >> 5;
    const int j = (blk * (TH / kWave) + wave) * 32 + (lane & 31);
    const int len = at_length(a, kb);
    const bool ok = j < len, busy = (blk * (TH / kWave) + wave) * 32 < len;
    const int64_t key = j < a.kv_len ? at_key(a, kb, j) : 0;

    typename Elem<T>::V8 kf[NC], vf[NC];
    at_load_row<T, DP, VEC>(kf, ok ? (const T*)a.k + kb * a.sk.b + hk * a.sk.h + key * a.sk.l : nullptr, a.d);
    at_load_row<T, DP, VEC>(vf, ok ? (const T*)a.v + kb * a.sv.b + hk * a.sv.h + key * a.sv.l : nullptr, a.d);
    f32x16 gk[NB], gv[NB];
    AtRange<T> range;
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) gk[db][i] = gv[db][i] = 0.0f;
    const int tiles = (a.rows + RT - 1) / RT, per = (tiles + a.splits - 1) / a.splits;
    const int t_end = blk * (TH / kWave) * 32 < len ? min(tiles, (sp + 1) * per) : 0;   // no allowed key: no rows
    AtTile<T, DP, RT, TH, VEC> tq, td;
    // Where chunk k's row stands, and how it goes RT rows on: a few additions, where at_row would divide. RT is so many batches,
    // queries and heads, each with one carry at most, however few queries a batch has. A row past the last stays on the last.
    constexpr int PER = decltype(tq)::kPer;
    int32_t row[PER], qi[PER], qh[PER];
    int64_t at_q[PER], at_d[PER], at_s[PER];
    float st[PER];
    const int G = (int)a.by_g.d, per_batch = (int)a.by_lg.d;
    const int step_b = RT / per_batch, step_i = RT % per_batch / G, step_h = RT % per_batch % G;
    const int64_t batch_s = (int64_t)a.heads * a.q_len;
    const int64_t step_q = step_b * a.sq.b + step_i * a.sq.l + step_h * a.sq.h;
    const int64_t step_d = step_b * a.sdo.b + step_i * a.sdo.l + step_h * a.sdo.h;
    const int64_t step_s = step_b * batch_s + step_i + (int64_t)step_h * a.q_len;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        row[k] = min(sp * per * RT + (tq.inside(k) ? tq.row(k) : 0), a.rows - 1);
        if (a.rows <= 0) continue;
        const AtRow at = at_row(a, kb, hk, row[k]);
        qi[k] = at.i;
        qh[k] = at.h - hk * G;
        at_q[k] = at_offset(a.sq, at);
        at_d[k] = at_offset(a.sdo, at);
        at_s[k] = at_stat(a, at);
    }
    auto fetch = [&]() {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            tq.load_row(k, (const T*)a.q + at_q[k], a.d);
            td.load_row(k, (const T*)a.dout + at_d[k], a.d);
            st[k] = (tq.col(k) == 0 ? a.lse : a.delta)[at_s[k]];   // the first chunk of a row brings lse, the others delta
            if (row[k] + RT < a.rows) {
                row[k] += RT;
                qi[k] += step_i;
                qh[k] += step_h;
                at_q[k] += step_q;
                at_d[k] += step_d;
                at_s[k] += step_s;
                if (qh[k] >= G) {   // the next query
                    qh[k] -= G;
                    qi[k] += 1;
                    at_q[k] += a.sq.l - G * a.sq.h;
                    at_d[k] += a.sdo.l - G * a.sdo.h;
                    at_s[k] += 1 - (int64_t)G * a.q_len;
                }
                if (qi[k] >= a.q_len) {   // the next batch
                    qi[k] -= a.q_len;
                    at_q[k] += a.sq.b - a.q_len * a.sq.l;
                    at_d[k] += a.sdo.b - a.q_len * a.sdo.l;
                    at_s[k] += batch_s - a.q_len;
                }
            }
        }
    };
    if (sp * per < t_end) fetch();
    for (int t = sp * per; t < t_end; ++t) {
        __syncthreads();
        tq.store(s_q, a.rows - t * RT, a.d);
        td.store(s_d, a.rows - t * RT, a.d);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const bool in = t * RT + tq.row(k) < a.rows;
            if (tq.inside(k) && tq.col(k) == 0) s_lse[tq.row(k)] = in ? at_lse2(st[k]) - at_p_shift<T>() : INFINITY;
            if (tq.inside(k) && tq.col(k) == 8) s_delta[tq.row(k)] = in ? -st[k] : 0.0f;
        }
        __syncthreads();
        if (t + 1 < t_end) fetch();
        if (!busy) continue;
#pragma unroll
        for (int rb = 0; rb < RT; rb += 32) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {   // dP - delta: the product starts from -delta
                const f32x4 de = *reinterpret_cast<const f32x4*>(s_delta + rb + k * 8 + h * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) dp[k * 4 + i] = de[i];
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = mma(at_rows<T, DP>(s_q, rb, c), kf[c], s);
                dp = mma(at_rows<T, DP>(s_d, rb, c), vf[c], dp);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(s_lse + rb + k * 8 + h * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k * 4 + i], a.c, -ls[i]));
                    s[k * 4 + i] = p;
                    dp[k * 4 + i] *= p;
                }
            }
            if constexpr (AtRange<T>::kOn) {
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] *= range.g;
                float f;
                if (range.lower(dp, &f)) {
                    dp *= f;
#pragma unroll
                    for (int db = 0; db < NB; ++db) gk[db] *= f;
                }
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const AtOperand<T, TWO> p(s, ks), ds(dp, ks);
#pragma unroll
                for (int db = 0; db < NB; ++db) {
                    gv[db] = p.product(at_cols<T, DP>(s_d, rb + ks * 16, db), gv[db]);
                    gk[db] = ds.product(at_cols<T, DP>(s_q, rb + ks * 16, db), gk[db]);
                }
            }
        }
    }
    if (!ok) {   // (a column of its own in every product, not masked before)
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) gk[db][i] = gv[db][i] = 0.0f;
    }
    const float undo_k = range.undo() * at_p_undo<T>();
    if (a.splits == 1) {
        const bool in = j < a.kv_len;
        at_store_row<T, DP>(in ? (T*)a.dk + kb * a.sdk.b + hk * a.sdk.h + key * a.sdk.l : nullptr, gk,
                            at_grad_scale(a, len) * undo_k, a.d, a.vec_out);
        at_store_row<T, DP>(in ? (T*)a.dv + kb * a.sdv.b + hk * a.sdv.h + key * a.sdv.l : nullptr, gv, at_p_undo<T>(), a.d,
                            a.vec_out);
    } else if (j < a.kv_len) {
        const int64_t all = (int64_t)(gridDim.x / (a.blocks * a.splits)) * a.kv_len;
        const int64_t pr = (2 * sp * all) + (int64_t)kvh * a.kv_len + j;
        at_store_row<float, DP>(a.part + pr * DP, gk, undo_k, DP, true);
        at_store_row<float, DP>(a.part + (pr + all) * DP, gv, at_p_undo<T>(), DP, true);
    }
}

// Sums the splits' partial gradients, always in the same order: dQ's rows (what 0), or dK's and dV's (what 1). One thread
// per four elements; with SG > 1, for many splits, SG of them take every SG-th split and are added up in LDS
// (64 splits of few results: 17 to 21 us by one thread each, 4.4 by eight).
template <class T, int SG>
__global__ __launch_bounds__(kAtThreads) void k_attend_sum(AtArgs a, int dp, int64_t all, int what) {
    __shared__ f32x4 s_x[SG > 1 ? kAtThreads : 1];
    __shared__ float s_delta[SG > 1 ? kAtThreads : 1];
    constexpr int per = kAtThreads / SG;
    const int g = (int)threadIdx.x / per;
    const int64_t id = (int64_t)blockIdx.x * per + (int)threadIdx.x % per;
    const int quads = dp / 4;
    const int64_t n = (what ? 2 : 1) * all;
    const int64_t pr = id / quads;
    const int e = (int)(id % quads) * 4;
    const bool in = pr < n && e < a.d;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    float delta = 0.0f;
    if (in) {
#pragma unroll 8
        for (int s = g; s < a.splits; s += SG) x += *reinterpret_cast<const f32x4*>(a.part + (s * n + pr) * dp + e);
        if (what == 0 && e == 0)
#pragma unroll 8
            for (int s = g; s < a.splits; s += SG) delta += a.part_ml[s * n + pr];
    }
    if constexpr (SG > 1) {
        s_x[threadIdx.x] = x;
        s_delta[threadIdx.x] = delta;
        __syncthreads();
        if (g == 0)
            for (int i = 1; i < SG; ++i) {
                x += s_x[threadIdx.x + i * per];
                delta += s_delta[threadIdx.x + i * per];
            }
    }
    if (!in || g > 0) return;
    if (what == 0) {
        const int kvh = (int)(pr / a.rows);
        const AtRow row = at_row(a, kvh / a.kv_heads, kvh % a.kv_heads, (int)(pr % a.rows));
        at_store4<T>((T*)a.dq + at_offset(a.sdq, row) + e, x * at_grad_scale(a, at_length(a, kvh / a.kv_heads)), a.d - e,
                     a.vec_out);
        if (e == 0) a.delta[at_stat(a, row)] = delta;
    } else {
        const bool is_v = pr >= all;
        const int64_t rest = is_v ? pr - all : pr;
        const int j = (int)(rest % a.kv_len), kvh = (int)(rest / a.kv_len);
        const AtHeads& st = is_v ? a.sdv : a.sdk;
        T* const p = (T*)(is_v ? a.dv : a.dk) + kvh / a.kv_heads * st.b + kvh % a.kv_heads * st.h +
                     at_key(a, kvh / a.kv_heads, j) * st.l;
        at_store4<T>(p + e, is_v ? x : x * at_grad_scale(a, at_length(a, kvh / a.kv_heads)), a.d - e, a.vec_out);
    }
}

// ---- host ----------------------------------------------------------------------------------

// Workgroups that run at a time, two per CU, and the most parts that the long axis of a launch with fewer is
// split into: as many as run together, since one more part for every workgroup would wait for a second round.
// With lengths or a mask, workgroups end at different times, and twice as many parts even that out.
constexpr int64_t kAtWorkgroups = 512;
constexpr int kAtSplits = 256;

// Results (elements of out; of dK) up to which P, and dS for dK, keep their bits by a second product. Rounded to a 16-bit
// type they leave an error as large as the results' own rounding, 1.4 times that together; over a large
// tensor it stays there, over a few results it may come to twice that.
constexpr int64_t kAtFewResults = 1 << 16;

static int at_splits(int64_t workgroups, int64_t tiles, bool uneven) {
    int64_t s = workgroups > 0 ? (uneven ? 2 : 1) * kAtWorkgroups / workgroups : 1;
    if (s > kAtSplits) s = kAtSplits;
    if (s > tiles) s = tiles;
    return (int)(s > 1 ? s : 1);
}

static int at_padded(int d) { return (d + 31) / 32 * 32; }

// Makes the list of the allowed keys in `temp` where there is a mask.
static int at_list(const tdgs_attention* a, AtArgs* r, void* temp, hipStream_t stream) {
    if (!a->kv_mask || a->kv_len == 0) return TDGS_OK;
    int32_t* const index = (int32_t*)temp;
    int32_t* const counts = index + (int64_t)a->kv_batch * a->kv_len;
    k_attend_list<<<(unsigned)a->kv_batch, kAtListThreads, 0, stream>>>(a->kv_mask, a->kv_mask_stride, *r, index, counts);
    TDGS_LAUNCHED();
    r->index = index;
    r->lengths = counts;
    return TDGS_OK;
}

// f(integral constant) for the padded head dimension.
template <class F>
static int with_padded(int dp, F&& f) {
    switch (dp) {
        case 32: return f(std::integral_constant<int, 32>{});
        case 64: return f(std::integral_constant<int, 64>{});
        case 96: return f(std::integral_constant<int, 96>{});
        default: return f(std::integral_constant<int, 128>{});
    }
}

static int at_forward_rows(int32_t dtype, int dp) {
    return with_dtype(dtype, [&](auto t) -> int {
        return with_padded(dp, [&](auto d) -> int { return AtForward<decltype(t), decltype(d)::value>::kRows; });
    });
}

// How the three launches are cut, from the sizes and whether there are lengths or a mask.
struct AtPlan {
    int64_t kvh, rows;   // kv heads over all kv batches; rows of each
    int dp, rows_f, tile;
    bool wide_k;
    int blocks_f, splits_f, blocks_q, splits_q, blocks_k, splits_k;
    size_t list_bytes, delta_bytes, forward_bytes, grad_bytes;   // (the first two within the last two)
};

static AtPlan at_plan(const tdgs_attention* a, bool uneven) {
    AtPlan p;
    p.kvh = (int64_t)a->kv_batch * a->kv_heads;
    p.rows = (int64_t)(a->kv_batch > 0 ? a->batch / a->kv_batch : 0) * a->q_len * (a->heads / a->kv_heads);
    p.dp = at_padded(a->head_dim);
    p.tile = a->dtype == TDGS_F32 ? 32 : 64;
    p.rows_f = at_forward_rows(a->dtype, p.dp);
    const int64_t key_tiles = ceil_div(a->kv_len, p.tile), row_tiles = ceil_div(p.rows, 32);
    p.blocks_f = (int)ceil_div(p.rows, p.rows_f);
    p.splits_f = at_splits(p.blocks_f * p.kvh, key_tiles, uneven);
    p.blocks_q = (int)ceil_div(p.rows, kAtWaves * 32);
    p.splits_q = at_splits(p.blocks_q * p.kvh, key_tiles, uneven);
    p.wide_k = a->dtype != TDGS_F32 && p.dp <= 64 && a->kv_len >= 512;   // (few idle wavefronts; registers to spare)
    p.blocks_k = (int)ceil_div(a->kv_len, p.wide_k ? kAtWide / 2 : kAtWaves * 32);
    p.splits_k = at_splits(p.blocks_k * p.kvh * (p.wide_k ? 2 : 1), p.wide_k ? ceil_div(p.rows, 64) : row_tiles, uneven);
    const size_t all_rows = (size_t)(p.kvh * p.rows), all_keys = (size_t)(p.kvh * a->kv_len);
    p.list_bytes = align_up((size_t)a->kv_batch * ((size_t)a->kv_len + 1) * sizeof(int32_t));
    p.delta_bytes = align_up(all_rows * sizeof(float));
    p.forward_bytes = (uneven ? p.list_bytes : 0) +
                      (p.splits_f > 1 ? align_up(p.splits_f * all_rows * (p.dp + 2) * sizeof(float)) : 0);
    const size_t q = p.splits_q > 1 ? p.splits_q * all_rows * (p.dp + 1) * sizeof(float) : 0;
    const size_t k = p.splits_k > 1 ? p.splits_k * 2 * all_keys * p.dp * sizeof(float) : 0;
    p.grad_bytes = (uneven ? p.list_bytes : 0) + p.delta_bytes + align_up(q > k ? q : k);
    return p;
}

static int at_check_view(const tdgs_heads* v, const char* name, const tdgs_attention* a, bool keys, bool written) {
    TDGS_REQUIRE(v->data != nullptr, "attention: %s is null", name);
    const size_t e = (size_t)dtype_size(a->dtype);
    TDGS_REQUIRE(aligned_to(v->data, e), "attention: %s is not aligned to its element type", name);
    const int64_t nb = keys ? a->kv_batch : a->batch, nl = keys ? a->kv_len : a->q_len, nh = keys ? a->kv_heads : a->heads;
    TDGS_REQUIRE(v->stride_b >= 0 && v->stride_l >= 0 && v->stride_h >= 0, "attention: %s has a negative stride", name);
    if (written)
        TDGS_REQUIRE((nb <= 1 || v->stride_b >= a->head_dim) && (nl <= 1 || v->stride_l >= a->head_dim) &&
                         (nh <= 1 || v->stride_h >= a->head_dim),
                     "attention: rows of %s overlap", name);
    return TDGS_OK;
}

static int at_check(const tdgs_attention* a) {
    TDGS_REQUIRE(a != nullptr, "attention: null arguments");
    TDGS_REQUIRE(known_dtype(a->dtype), "attention: unknown element type %d", a->dtype);
    TDGS_REQUIRE(a->batch >= 0 && a->q_len >= 0 && a->kv_len >= 0, "attention: negative size");
    TDGS_REQUIRE(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0,
                 "attention: %d query heads do not divide among %d kv heads", a->heads, a->kv_heads);
    TDGS_REQUIRE(a->kv_batch == a->batch || a->kv_batch == 1, "attention: kv batch %d is neither the batch %d nor 1",
                 a->kv_batch, a->batch);
    TDGS_REQUIRE(a->head_dim >= 1 && a->head_dim <= 128, "attention: head dimension %d is not in 1 to 128", a->head_dim);
    TDGS_REQUIRE(a->scale > 0.0f && a->scale < INFINITY, "attention: the scale must be positive and finite");
    const int64_t g = a->heads / a->kv_heads;
    TDGS_REQUIRE((int64_t)a->batch * a->q_len <= INT32_MAX / g - 256, "attention: too many queries for one kv head");
    TDGS_REQUIRE((int64_t)a->batch * a->heads <= INT32_MAX / (a->q_len / 128 + 1) / kAtSplits, "attention: too many heads");
    TDGS_REQUIRE(a->kv_len <= INT32_MAX - 256, "attention: too many keys");
    TDGS_REQUIRE((int64_t)a->kv_batch * a->kv_heads <= INT32_MAX / (a->kv_len / 128 + 1) / kAtSplits, "attention: too many kv heads");
    return TDGS_OK;
}

static AtHeads at_strides(const tdgs_heads& v) { return {v.stride_b, v.stride_l, v.stride_h}; }

template <class T>
static int at_sum(const AtArgs& r, int dp, int64_t all, int what, hipStream_t stream) {
    const int64_t items = (what ? 2 : 1) * all * (dp / 4);
    if (r.splits >= 16) k_attend_sum<T, 8><<<(unsigned)ceil_div(items, kAtThreads / 8), kAtThreads, 0, stream>>>(r, dp, all, what);
    else k_attend_sum<T, 1><<<(unsigned)ceil_div(items, kAtThreads), kAtThreads, 0, stream>>>(r, dp, all, what);
    TDGS_LAUNCHED();
    return TDGS_OK;
}

// Whether rows of the view start on 16 bytes.
static bool at_rows_aligned(const tdgs_heads& v, int64_t e) {
    return aligned_to(v.data, 16) && v.stride_b * e % 16 == 0 && v.stride_l * e % 16 == 0 && v.stride_h * e % 16 == 0;
}

static AtArgs at_args(const tdgs_attention* a, const AtPlan& p) {
    AtArgs r = {};
    const int64_t e = dtype_size(a->dtype);
    r.q = a->q.data;
    r.k = a->k.data;
    r.v = a->v.data;
    r.o = r.out = a->out.data;
    r.sq = at_strides(a->q);
    r.sk = at_strides(a->k);
    r.sv = at_strides(a->v);
    r.so = at_strides(a->out);
    r.lengths = a->kv_lengths;
    r.lse = a->lse;
    r.q_len = a->q_len;
    r.kv_len = a->kv_len;
    r.heads = a->heads;
    r.kv_heads = a->kv_heads;
    r.d = a->head_dim;
    r.rows = (int32_t)p.rows;
    r.group_batches = a->batch / a->kv_batch;
    r.scale = a->scale;
    r.c = a->scale * kLog2e;
    const uint32_t g = (uint32_t)(a->heads / a->kv_heads);
    r.by_g = FastDiv(g);
    r.by_lg = FastDiv(p.rows > 0 ? g * (uint32_t)a->q_len : 1);   // (no rows: never divided by)
    r.vec_out = a->head_dim % 8 == 0 && at_rows_aligned(a->out, e);
    return r;
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

size_t tdgs_cross_attention_temp_bytes(const tdgs_attention* a, int32_t grad) {
    if (at_check(a) != TDGS_OK || a->kv_batch == 0) return 0;
    size_t bytes = 0;
    for (int uneven = 0; uneven < 2; ++uneven) {
        const AtPlan p = at_plan(a, uneven != 0);
        const size_t b = grad && p.grad_bytes > p.forward_bytes ? p.grad_bytes : p.forward_bytes;
        if (b > bytes) bytes = b;
    }
    return bytes;
}

int tdgs_cross_attention(void* stream_, const tdgs_attention* a) {
    TDGS_TRY(at_check(a));
    if (a->batch == 0 || a->q_len == 0) return TDGS_OK;
    TDGS_TRY(at_check_view(&a->q, "q", a, false, false));
    TDGS_TRY(at_check_view(&a->out, "out", a, false, true));
    if (a->kv_len > 0) {
        TDGS_TRY(at_check_view(&a->k, "k", a, true, false));
        TDGS_TRY(at_check_view(&a->v, "v", a, true, false));
    }
    const bool uneven = a->kv_lengths || a->kv_mask;
    const AtPlan p = at_plan(a, uneven);
    TDGS_REQUIRE(p.forward_bytes == 0 || (a->temp && a->temp_bytes >= p.forward_bytes && aligned_to(a->temp, 16)),
                 "attention: scratch of %zu bytes, %zu needed", a->temp ? a->temp_bytes : (size_t)0, p.forward_bytes);
    hipStream_t stream = (hipStream_t)stream_;
    AtArgs r = at_args(a, p);
    r.blocks = p.blocks_f;
    r.splits = p.splits_f;
    const int64_t all = p.kvh * p.rows;
    TDGS_TRY(at_list(a, &r, a->temp, stream));
    if (p.splits_f > 1) {
        r.part = (float*)((char*)a->temp + (uneven ? p.list_bytes : 0));
        r.part_ml = r.part + p.splits_f * all * p.dp;
    }
    const int64_t e = dtype_size(a->dtype);
    const bool vec = a->head_dim % 8 == 0 && at_rows_aligned(a->q, e) &&
                     (a->kv_len == 0 || (at_rows_aligned(a->k, e) && at_rows_aligned(a->v, e)));
    const unsigned grid = (unsigned)(p.kvh * p.splits_f * p.blocks_f);
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        TDGS_TRY(with_padded(p.dp, [&](auto dp) -> int {
            constexpr int DP = decltype(dp)::value, TH = AtForward<T, DP>::kThreads;
            auto launch = [&](auto two) {
                constexpr bool TWO = decltype(two)::value;
                if (vec && !r.index && !TWO) k_attend<T, DP, true, false, false><<<grid, TH, 0, stream>>>(r);
                else if (vec) k_attend<T, DP, true, true, TWO><<<grid, TH, 0, stream>>>(r);
                else k_attend<T, DP, false, true, TWO><<<grid, TH, 0, stream>>>(r);
            };
            if (sizeof(T) == 2 && all * a->head_dim <= kAtFewResults) launch(std::integral_constant<bool, sizeof(T) == 2>{});
            else launch(std::false_type{});
            TDGS_LAUNCHED();
            return TDGS_OK;
        }));
        if (p.splits_f > 1) {
            const int per = kAtThreads / (p.dp / 4);   // rows per workgroup
            if (p.splits_f >= 8) k_attend_join<T, 8><<<(unsigned)ceil_div(all, per / 8), kAtThreads, 0, stream>>>(r, p.dp, all);
            else k_attend_join<T, 1><<<(unsigned)ceil_div(all, per), kAtThreads, 0, stream>>>(r, p.dp, all);
            TDGS_LAUNCHED();
        }
        return TDGS_OK;
    });
}

int tdgs_cross_attention_grad(void* stream_, const tdgs_attention* a, const tdgs_attention_grads* g) {
    TDGS_TRY(at_check(a));
    TDGS_REQUIRE(g != nullptr, "attention: null gradients");
    // without queries dk and dv are zero, and written (a batch of none may share states)
    const bool queries = a->batch > 0 && a->q_len > 0;
    const bool keys = a->kv_batch > 0 && a->kv_len > 0, key_grads = keys && (g->dk.data || g->dv.data);
    if (!queries && !key_grads) return TDGS_OK;
    if (queries) {
        TDGS_TRY(at_check_view(&a->q, "q", a, false, false));
        TDGS_TRY(at_check_view(&a->out, "out", a, false, false));
        TDGS_TRY(at_check_view(&g->dout, "dout", a, false, false));
        TDGS_TRY(at_check_view(&g->dq, "dq", a, false, true));
        TDGS_REQUIRE(a->lse != nullptr, "attention: the gradient needs the forward call's lse");
    }
    if (keys) {
        TDGS_TRY(at_check_view(&a->k, "k", a, true, false));
        TDGS_TRY(at_check_view(&a->v, "v", a, true, false));
    }
    if (key_grads) {
        TDGS_TRY(at_check_view(&g->dk, "dk", a, true, true));
        TDGS_TRY(at_check_view(&g->dv, "dv", a, true, true));
    }
    const bool uneven = a->kv_lengths || a->kv_mask;
    const AtPlan p = at_plan(a, uneven);
    TDGS_REQUIRE(p.grad_bytes == 0 || (a->temp && a->temp_bytes >= p.grad_bytes && aligned_to(a->temp, 16)),
                 "attention: scratch of %zu bytes, the gradient needs %zu", a->temp ? a->temp_bytes : (size_t)0,
                 p.grad_bytes);
    hipStream_t stream = (hipStream_t)stream_;
    AtArgs r = at_args(a, p);
    const int64_t e = dtype_size(a->dtype);
    r.dout = g->dout.data;
    r.dq = g->dq.data;
    r.dk = g->dk.data;
    r.dv = g->dv.data;
    r.sdo = at_strides(g->dout);
    r.sdq = at_strides(g->dq);
    r.sdk = at_strides(g->dk);
    r.sdv = at_strides(g->dv);
    const bool vec = r.vec_out && at_rows_aligned(a->q, e) && at_rows_aligned(g->dout, e) && at_rows_aligned(a->k, e) &&
                     at_rows_aligned(a->v, e);
    r.vec_out = a->head_dim % 8 == 0 && at_rows_aligned(g->dq, e) && at_rows_aligned(g->dk, e) && at_rows_aligned(g->dv, e);
    TDGS_TRY(at_list(a, &r, a->temp, stream));
    r.delta = (float*)((char*)a->temp + (uneven ? p.list_bytes : 0));
    r.part = (float*)((char*)r.delta + p.delta_bytes);
    const int64_t all_rows = p.kvh * p.rows, all_keys = p.kvh * a->kv_len;
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        return with_padded(p.dp, [&](auto dp) -> int {
            constexpr int DP = decltype(dp)::value;
            if (queries) {
                r.blocks = p.blocks_q;
                r.splits = p.splits_q;
                r.part_ml = r.part + p.splits_q * all_rows * DP;
                const unsigned grid = (unsigned)(p.kvh * p.splits_q * p.blocks_q);
                if (vec && !r.index) k_attend_dq<T, DP, true, false><<<grid, kAtThreads, 0, stream>>>(r);
                else if (vec) k_attend_dq<T, DP, true, true><<<grid, kAtThreads, 0, stream>>>(r);
                else k_attend_dq<T, DP, false, true><<<grid, kAtThreads, 0, stream>>>(r);
                TDGS_LAUNCHED();
                if (p.splits_q > 1) {
                    TDGS_TRY(at_sum<T>(r, DP, all_rows, 0, stream));
                }
            }
            if (key_grads) {
                r.blocks = p.blocks_k;
                r.splits = p.splits_k;
                const unsigned grid = (unsigned)(p.kvh * p.splits_k * p.blocks_k);
                const bool few = sizeof(T) == 2 && all_keys * a->head_dim <= kAtFewResults;
                auto launch = [&](auto th, auto two) {
                    constexpr int TH = decltype(th)::value;
                    constexpr bool TWO = decltype(two)::value;
                    if (vec) k_attend_dkv<T, DP, TH, true, TWO><<<grid, TH, 0, stream>>>(r);
                    else k_attend_dkv<T, DP, TH, false, TWO><<<grid, TH, 0, stream>>>(r);
                };
                using Narrow = std::integral_constant<int, kAtThreads>;
                using Two = std::integral_constant<bool, sizeof(T) == 2>;
                if constexpr (sizeof(T) == 2 && DP <= 64) {
                    using Wide = std::integral_constant<int, kAtWide>;
                    if (p.wide_k && few) launch(Wide{}, Two{});
                    else if (p.wide_k) launch(Wide{}, std::false_type{});
                    else if (few) launch(Narrow{}, Two{});
                    else launch(Narrow{}, std::false_type{});
                } else {
                    if (few) launch(Narrow{}, Two{});
                    else launch(Narrow{}, std::false_type{});
                }
                TDGS_LAUNCHED();
                if (p.splits_k > 1) {
                    TDGS_TRY(at_sum<T>(r, DP, all_keys, 1, stream));
                }
            }
            return TDGS_OK;
        });
    });
}

}  // extern "C"
