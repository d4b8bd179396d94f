// linear.hip — linear layers with bias, activation and residual, forward and backward, on the matrix cores.
//
// Three products: z = x W, dx = dz W^T and dW = x^T dz. All are C (P x Q) = A (P x R) B (R x Q) with C's rows contiguous;
// what differs is whether an operand's depth r or its items (p or q) are contiguous in memory. A weight matrix
// may lie either way round; its gradient is computed as the transposed product where that is asked for.
//
// A workgroup holds a tile of C in registers, as 32x32 blocks (elem.hpp) of C^T, so that a lane has four
// neighbouring q of a row p. Tiles of A and B go from memory to registers to LDS as they lie in memory; operands
// whose items are contiguous are transposed by the reads from LDS. Where a row's end is no multiple of 16 bytes,
// its last chunk is loaded from the row's last 16 bytes and shifted into place, so that nothing is
// read past a row. The depth is split where there are few tiles, and partial sums of 32 bits joined by a
// second kernel, in the order of the splits.
//
// The epilogue turns blocks through LDS, so that 16 bytes of a row are one lane's, and adds the bias, keeps z where
// wanted, applies the activation and adds the residual, all in 32 bits; only what is stored is rounded.
#include "internal.hpp"
#include "elem.hpp"
#include "activation.hpp"

namespace tdgs {

struct LnMatrix {
    void* p;
    int64_t stride;
};

struct LnArgs {
    LnMatrix a, b;
    int32_t P, Q, R;
    int32_t tiles_p, tiles_q, splits, steps;   // steps: of the depth, per split
    float* part;              // splits x P x part_q, where splits > 1
    int32_t part_q;
    int32_t act;
    LnMatrix out, residual, pre;
    const void* bias;
    const float* scale;       // out = act(*scale C + ..); null: 1
};

// Elements of 16 bytes.
template <class T>
constexpr int ln_chunk() { return 16 / (int)sizeof(T); }
// Elements between LDS rows. Depth contiguous: 16 bytes of padding, and a read of 16 rows covers the banks once. Items
// contiguous: rows 16 banks apart for the transposing reads of four rows, four banks apart for single floats,
// whose two halves are eight rows apart.
template <class T, bool DEPTH, int N>
constexpr int ln_pitch() { return N + (DEPTH || sizeof(T) == 4 ? ln_chunk<T>() : 32); }

// A tile of MAJ memory rows x MIN elements on its way to LDS, by TH threads.
template <class T, int MAJ, int MIN, int TH, int PITCH>
struct LnTile {
    static constexpr int C = ln_chunk<T>();
    static constexpr int kChunks = MAJ * MIN / C;
    static constexpr int kPer = (kChunks + TH - 1) / TH;
    typedef uint32_t U4 __attribute__((ext_vector_type(4)));
    typedef T Ca __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    U4 r[kPer];
    __device__ __forceinline__ static int chunk(int k) { return (int)threadIdx.x + k * TH; }
    __device__ __forceinline__ static bool inside(int k) { return kChunks % TH == 0 || chunk(k) < kChunks; }
    __device__ __forceinline__ static int row(int k) { return inside(k) ? chunk(k) / (MIN / C) : 0; }
    __device__ __forceinline__ static int col(int k) { return inside(k) ? chunk(k) % (MIN / C) * C : 0; }
    // The tile at p, of whose rows `maj` > 0 and of whose elements `min` > 0 exist; the memory row holds C elements or more.
    __device__ __forceinline__ void load(const T* p, int64_t stride, int maj, int min) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int y = row(k) < maj ? row(k) : maj - 1, x = col(k) + C <= min ? col(k) : min - C;
            r[k] = __builtin_bit_cast(U4, *reinterpret_cast<const Ca*>(p + y * stride + x));
        }
    }
    // The same by single elements, for memory rows of fewer than C of them.
    __device__ __forceinline__ void load_narrow(const T* p, int64_t stride, int maj, int min) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int y = row(k) < maj ? row(k) : maj - 1;
            T e[C];
#pragma unroll
            for (int i = 0; i < C; ++i) e[i] = col(k) + i < min ? p[y * stride + col(k) + i] : (T)0.0f;
            r[k] = __builtin_bit_cast(U4, e);
        }
    }
    template <bool NARROW>
    __device__ __forceinline__ void store(T* lds, int maj, int min) {
        if (!NARROW && min < MIN) {   // chunks across the rows' end
            const int rest = min % C;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                if (col(k) >= min) r[k] = (U4)0;
                else if (col(k) + C > min) r[k] = shift_down(r[k], (C - rest) * (int)sizeof(T) * 8);
            }
        }
        if (maj < MAJ) {
#pragma unroll
            for (int k = 0; k < kPer; ++k)
                if (row(k) >= maj) r[k] = (U4)0;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (inside(k)) *reinterpret_cast<U4*>(lds + row(k) * PITCH + col(k)) = r[k];
    }
    // The 128 bits shifted down by `bits` of 1 to 127, zeros from above.
    __device__ __forceinline__ static U4 shift_down(U4 v, int bits) {
        uint64_t lo = v[0] | (uint64_t)v[1] << 32, hi = v[2] | (uint64_t)v[3] << 32;
        if (bits >= 64) {
            lo = hi;
            hi = 0;
            bits -= 64;
        }
        if (bits) {
            lo = lo >> bits | hi << (64 - bits);
            hi >>= bits;
        }
        return U4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
};

// An operand of a 32x32 product: items base.. of the tile, depth chunk c. Slot (l / 32) * 8 + i is depth 16 c + that.
template <class T, bool DEPTH, int PITCH>
__device__ __forceinline__ typename Elem<T>::V8 ln_operand(const T* lds, int base, int c) {
    const int l = (int)__lane_id();
    if constexpr (DEPTH) {
        return *reinterpret_cast<const typename Elem<T>::V8a*>(lds + (base + (l & 31)) * PITCH + c * 16 + (l >> 5) * 8);
    } else if constexpr (sizeof(T) == 4) {
        typename Elem<T>::V8 r;
        const T* p = lds + (c * 16 + (l >> 5) * 8) * PITCH + base + (l & 31);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = p[i * PITCH];
        return r;
    } else {   // 16 lanes give the addresses of 4 rows x 16 items, and each gets one item
        typedef short s4 __attribute__((ext_vector_type(4)));
        const T* p = lds + (c * 16 + (l >> 5) * 8 + ((l & 15) >> 2)) * PITCH + base + ((l >> 4) & 1) * 16 + (l & 3) * 4;
        typedef __attribute__((address_space(3))) s4* lp;
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * PITCH));
        return __builtin_bit_cast(typename Elem<T>::V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

template <class T>
struct LnVec {   // up to eight neighbouring elements of a row
    typedef T Va __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    __device__ __forceinline__ static void load(const T* p, int n, float (&f)[8]) {
        if (n >= 8) {
            const Va v = *reinterpret_cast<const Va*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = i < n ? (float)p[i] : 0.0f;
        }
    }
    __device__ __forceinline__ static void store(T* p, int n, const float (&f)[8]) {
        if (n >= 8) {
            Va v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (T)f[i];
            *reinterpret_cast<Va*>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = (T)f[i];
        }
    }
};

template <int ACT>
__device__ __forceinline__ void ln_act8(float (&v)[8]) {
    float none;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value<ACT, false>(v[i], &none);
}
__device__ __forceinline__ void ln_activate(int act, float (&v)[8]) {
    switch (act) {
        case TDGS_ACT_SILU: ln_act8<TDGS_ACT_SILU>(v); break;
        case TDGS_ACT_GELU: ln_act8<TDGS_ACT_GELU>(v); break;
        case TDGS_ACT_RELU: ln_act8<TDGS_ACT_RELU>(v); break;
        default: break;
    }
}

// The end of n (1 to 8) neighbouring results q.. of row p.
template <class T>
__device__ __forceinline__ void ln_finish(const LnArgs& a, float scale, int64_t p, int q, int n, float (&v)[8]) {
    if (a.scale) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= scale;
    }
    if (a.bias) {
        float b[8];
        LnVec<T>::load((const T*)a.bias + q, n, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    if (a.pre.p) LnVec<T>::store((T*)a.pre.p + p * a.pre.stride + q, n, v);
    ln_activate(a.act, v);
    if (a.residual.p) {
        float r[8];
        LnVec<T>::load((const T*)a.residual.p + p * a.residual.stride + q, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    LnVec<T>::store((T*)a.out.p + p * a.out.stride + q, n, v);
}

// A kernel's tile: BP x BQ of C by WP x WQ wavefronts, BK deep. AD, BD: whether the operands' depth is contiguous in
// memory. NARROW: an operand has memory rows of fewer elements than a chunk.
template <class T_, int BP_, int BQ_, int WP_, int WQ_, int BK_, bool AD_, bool BD_, bool NARROW_>
struct LnShape {
    typedef T_ T;
    static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, BK = BK_;
    static constexpr bool AD = AD_, BD = BD_, NARROW = NARROW_;
    static constexpr int TH = WP * WQ * kWave;
    static constexpr int NP = BP / WP / 32, NQ = BQ / WQ / 32;   // blocks per wavefront
    static constexpr int AMAJ = AD ? BP : BK, AMIN = AD ? BK : BP;
    static constexpr int BMAJ = BD ? BQ : BK, BMIN = BD ? BK : BQ;
    static constexpr int APITCH = ln_pitch<T, AD, AMIN>(), BPITCH = ln_pitch<T, BD, BMIN>();
    static constexpr int kA = AMAJ * APITCH, kB = BMAJ * BPITCH;         // elements of a stage
    static constexpr int kTurn = BQ / WQ + 4;                            // floats between rows of a turned block
    static constexpr size_t kStages = 2 * (size_t)(kA + kB) * sizeof(T);
    static constexpr size_t kEnd = (size_t)WP * WQ * 32 * kTurn * sizeof(float);
    static constexpr size_t kLds = kStages > kEnd ? kStages : kEnd;
};

template <class S>
__global__ __launch_bounds__(S::TH) void k_linear(LnArgs a) {
    using T = typename S::T;
    __shared__ __attribute__((aligned(16))) char s_mem[S::kLds];
    T* const s = reinterpret_cast<T*>(s_mem);
    const int wave = (int)threadIdx.x / kWave, lane = (int)__lane_id();
    const int wp = wave / S::WQ * (S::BP / S::WP), wq = wave % S::WQ * (S::BQ / S::WQ);
    const int item = xcd_band_item(blockIdx.x, gridDim.x);
    const int tiles = a.tiles_p * a.tiles_q, split = item / tiles, tile = item - split * tiles;
    const int p0 = tile / a.tiles_q * S::BP, q0 = tile % a.tiles_q * S::BQ;
    const int r_begin = split * a.steps * S::BK, r_end = min(a.R, r_begin + a.steps * S::BK);
    const int steps = (r_end - r_begin + S::BK - 1) / S::BK;

    f32x16 acc[S::NP][S::NQ];
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
        for (int j = 0; j < S::NQ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    LnTile<T, S::AMAJ, S::AMIN, S::TH, S::APITCH> ta;
    LnTile<T, S::BMAJ, S::BMIN, S::TH, S::BPITCH> tb;
    const int np = min(S::BP, a.P - p0), nq = min(S::BQ, a.Q - q0);
    auto load = [&](int step) {
        const int r0 = r_begin + step * S::BK, nr = r_end - r0;
        const T* const pa = (const T*)a.a.p + (S::AD ? p0 * a.a.stride + r0 : r0 * a.a.stride + p0);
        const T* const pb = (const T*)a.b.p + (S::BD ? q0 * a.b.stride + r0 : r0 * a.b.stride + q0);
        if constexpr (S::NARROW) {
            ta.load_narrow(pa, a.a.stride, S::AD ? np : nr, S::AD ? nr : np);
            tb.load_narrow(pb, a.b.stride, S::BD ? nq : nr, S::BD ? nr : nq);
        } else {
            ta.load(pa, a.a.stride, S::AD ? np : nr, S::AD ? nr : np);
            tb.load(pb, a.b.stride, S::BD ? nq : nr, S::BD ? nr : nq);
        }
    };
    auto store = [&](int step) {
        const int nr = r_end - r_begin - step * S::BK;
        T* const at = s + (step & 1) * (S::kA + S::kB);
        ta.template store<S::NARROW>(at, S::AD ? np : nr, S::AD ? nr : np);
        tb.template store<S::NARROW>(at + S::kA, S::BD ? nq : nr, S::BD ? nr : nq);
    };
    if (steps > 0) {
        load(0);
        store(0);
        if (steps > 1) load(1);
    }
    for (int step = 0; step < steps; ++step) {
        __syncthreads();
        if (step + 1 < steps) store(step + 1);
        if (step + 2 < steps) load(step + 2);
        const T* const la = s + (step & 1) * (S::kA + S::kB);
        const T* const lb = la + S::kA;
#pragma unroll
        for (int c = 0; c < S::BK / 16; ++c) {
            typename Elem<T>::V8 fa[S::NP], fb[S::NQ];
#pragma unroll
            for (int i = 0; i < S::NP; ++i) fa[i] = ln_operand<T, S::AD, S::APITCH>(la, wp + i * 32, c);
#pragma unroll
            for (int j = 0; j < S::NQ; ++j) fb[j] = ln_operand<T, S::BD, S::BPITCH>(lb, wq + j * 32, c);
#pragma unroll
            for (int i = 0; i < S::NP; ++i)
#pragma unroll
                for (int j = 0; j < S::NQ; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
        }
    }
    __syncthreads();

    // 32 rows at a time through the wavefront's own part of LDS
    float* const turn = reinterpret_cast<float*>(s_mem) + wave * 32 * S::kTurn;
    const float scale = a.scale ? *a.scale : 1.0f;
    constexpr int kPerRow = S::NQ * 4;          // lanes of a row, with eight results each
    constexpr int kRows = kWave / kPerRow;
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
#pragma unroll
        for (int j = 0; j < S::NQ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
                *reinterpret_cast<f32x4*>(turn + (lane & 31) * S::kTurn + j * 32 + g * 8 + (lane >> 5) * 4) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += kRows) {
            const int y = r0 + lane / kPerRow, x = lane % kPerRow * 8, p = p0 + wp + i * 32 + y, q = q0 + wq + x;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(turn + y * S::kTurn + x);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(turn + y * S::kTurn + x + 4);
            if (p >= a.P || q >= a.Q) continue;
            if (a.part) {
                f32x4* const o = reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.P + p) * a.part_q + q);
                o[0] = lo;
                o[1] = hi;
            } else {
                float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                ln_finish<T>(a, scale, p, q, min(8, a.Q - q), v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Joins the splits' sums, eight neighbouring results per thread.
constexpr int kLnThreads = 256;
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_join(LnArgs a) {
    const int chunks = a.part_q / 8;
    const int64_t i = (int64_t)blockIdx.x * kLnThreads + threadIdx.x;
    if (i >= (int64_t)a.P * chunks) return;
    const int64_t p = i / chunks;
    const int q = (int)(i - p * chunks) * 8;
    const float scale = a.scale ? *a.scale : 1.0f;
    float v[8] = {};
    for (int s = 0; s < a.splits; ++s) {
        const f32x4* const o = reinterpret_cast<const f32x4*>(a.part + ((int64_t)s * a.P + p) * a.part_q + q);
        const f32x4 lo = o[0], hi = o[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += lo[e];
            v[e + 4] += hi[e];
        }
    }
    ln_finish<T>(a, scale, p, q, min(8, a.Q - q), v);
}

// ---- the gradient's elementwise part: dz = dout act'(z), and its columns' sums ------------------

struct LnGradArgs {
    LnMatrix dout, pre, dz;     // dz null: not wanted
    int64_t rows;
    int32_t n, act, blocks;
    int64_t per;                // rows per workgroup
    float* sums;                // blocks x n; null: not wanted
    const float* top;           // float16: partial maxima of |dout|; null: dz is not scaled
    int32_t tops;
    float* scale;               // what undoes dz's power of two
};

// The largest |dout| of each workgroup's share (float16).
constexpr int kLnTops = 256;
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_top(LnGradArgs a, float* top) {
    __shared__ float s[kLnThreads / kWave];
    float m = 0.0f;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* const p = (const T*)a.dout.p + r * a.dout.stride;
        for (int q = (int)threadIdx.x * 8; q < a.n; q += kLnThreads * 8) {
            float v[8];
            LnVec<T>::load(p + q, min(8, a.n - q), v);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
        }
    }
    for (int w = kWave / 2; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, kWave));
    if (__lane_id() == 0) s[threadIdx.x / kWave] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLnThreads / kWave; ++w) m = fmaxf(m, s[w]);
        top[blockIdx.x] = m;
    }
}

// The power of two that brings a tensor whose largest value is m to 2^14, so that its products with act' (below 1.2)
// stay in half's range.
__device__ __forceinline__ float ln_range(float m) {
    if (!(m > 0.0f)) return 1.0f;
    const int e = min((int)(__builtin_bit_cast(uint32_t, m) >> 23) - 127, 16);   // (infinity: as the largest half)
    return __builtin_bit_cast(float, (uint32_t)(14 - e + 127) << 23);
}

// Workgroup (x, y): 64 chunks of eight columns by four rows at a time, of the y-th run of rows.
template <class T, int ACT>
__global__ __launch_bounds__(kLnThreads) void k_linear_dz(LnGradArgs a) {
    __shared__ float s[kLnThreads / kWave][kWave * 8];
    const int lane = (int)__lane_id(), wave = (int)threadIdx.x / kWave, q = ((int)blockIdx.x * kWave + lane) * 8;
    float up = 1.0f;
    if (a.top) {
        float m = a.top[threadIdx.x % a.tops];
        for (int w = kWave / 2; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, kWave));
        if (lane == 0) s[wave][0] = m;
        __syncthreads();
        for (int w = 0; w < kLnThreads / kWave; ++w) m = fmaxf(m, s[w][0]);
        __syncthreads();
        up = ln_range(m);
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.scale = 1.0f / up;
    }
    const int n = a.n - q;
    float sum[8] = {};
    if (n > 0) {
        const int64_t end = min(a.rows, (blockIdx.y + (int64_t)1) * a.per);
        for (int64_t r = blockIdx.y * a.per + wave; r < end; r += kLnThreads / kWave) {
            float d[8];
            LnVec<T>::load((const T*)a.dout.p + r * a.dout.stride + q, n, d);
            if constexpr (ACT != TDGS_ACT_IDENTITY) {
                float z[8], slope;
                LnVec<T>::load((const T*)a.pre.p + r * a.pre.stride + q, n, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    act_value<ACT, true>(z[i], &slope);
                    d[i] *= slope;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += d[i];
            if (a.dz.p) {
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= up;
                LnVec<T>::store((T*)a.dz.p + r * a.dz.stride + q, n, d);
            }
        }
    }
    if (!a.sums) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[wave][lane * 8 + i] = sum[i];
    __syncthreads();
    for (int c = threadIdx.x; c < kWave * 8; c += kLnThreads) {
        const int col = (int)blockIdx.x * kWave * 8 + c;
        if (col >= a.n) break;
        float x = 0.0f;
        for (int w = 0; w < kLnThreads / kWave; ++w) x += s[w][c];
        a.sums[(int64_t)blockIdx.y * a.n + col] = x;
    }
}

// dbias from the runs' sums: eight columns per workgroup.
constexpr int kLnBiasCols = 8;
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_dbias(const float* __restrict__ sums, int blocks, int n, T* dbias) {
    __shared__ float s[kLnThreads / kLnBiasCols][kLnBiasCols + 1];
    const int x = (int)threadIdx.x % kLnBiasCols, y = (int)threadIdx.x / kLnBiasCols, c = blockIdx.x * kLnBiasCols + x;
    float v = 0.0f;
    if (c < n)
        for (int b = y; b < blocks; b += kLnThreads / kLnBiasCols) v += sums[(int64_t)b * n + c];
    s[y][x] = v;
    __syncthreads();
    if (y != 0 || c >= n) return;
    for (int i = 1; i < kLnThreads / kLnBiasCols; ++i) v += s[i][x];
    dbias[c] = (T)v;
}

// What is zero without rows (dweight and dbias).
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_zero(T* p, int64_t rows, int cols, int64_t stride) {
    const int64_t i = (int64_t)blockIdx.x * kLnThreads + threadIdx.x;
    if (i < rows * cols) p[i / cols * stride + i % cols] = (T)0.0f;
}

// ---- host ----------------------------------------------------------------------------------

// Workgroups that fill the card, and the least depth (in steps) of a split.
constexpr int64_t kLnWorkgroups = 512;
constexpr int kLnLeastSteps = 8;

template <class T>
constexpr int ln_depth() { return sizeof(T) == 4 ? 16 : 32; }

// How a product is cut.
struct LnPlan {
    bool large;        // 128 x 128 tiles, 64 x 64 otherwise
    int tiles_p, tiles_q, splits, steps, part_q;
    size_t bytes;
};

static LnPlan ln_plan(int32_t dtype, int64_t P, int64_t Q, int64_t R) {
    LnPlan p;
    const int depth = dtype == TDGS_F32 ? ln_depth<float>() : ln_depth<bf16>();
    p.large = ceil_div(P, 128) * ceil_div(Q, 128) >= 256 || (P > 64 && Q > 64 && R >= 4096);
    const int side = p.large ? 128 : 64;
    p.tiles_p = (int)ceil_div(P, side);
    p.tiles_q = (int)ceil_div(Q, side);
    const int64_t tiles = (int64_t)p.tiles_p * p.tiles_q, steps = ceil_div(R, depth);
    int64_t splits = tiles > 0 ? kLnWorkgroups / tiles : 1;
    if (splits > steps / kLnLeastSteps) splits = steps / kLnLeastSteps;
    if (splits < 1) splits = 1;
    p.steps = (int)ceil_div(steps, splits);
    p.splits = (int)(p.steps > 0 ? ceil_div(steps, p.steps) : 1);
    p.part_q = (int)(ceil_div(Q, 8) * 8);
    p.bytes = p.splits > 1 ? align_up((size_t)p.splits * P * p.part_q * sizeof(float)) : 0;
    return p;
}

// C = A B, with what follows it in `r`.
template <class T, bool AD, bool BD>
static int ln_product(LnArgs r, const LnPlan& p, void* temp, hipStream_t stream) {
    r.tiles_p = p.tiles_p;
    r.tiles_q = p.tiles_q;
    r.splits = p.splits;
    r.steps = p.steps;
    r.part_q = p.part_q;
    r.part = p.splits > 1 ? (float*)temp : nullptr;
    const int64_t grid = (int64_t)p.tiles_p * p.tiles_q * p.splits;
    TDGS_REQUIRE(grid <= INT32_MAX, "linear: too many tiles");
    constexpr int C = ln_chunk<T>(), D = ln_depth<T>();
    const bool narrow = (AD ? r.R : r.P) < C || (BD ? r.R : r.Q) < C;
    auto launch = [&](auto shape) {
        using S = decltype(shape);
        k_linear<S><<<(unsigned)grid, S::TH, 0, stream>>>(r);
    };
    if (p.large && !narrow) launch(LnShape<T, 128, 128, 2, 2, D, AD, BD, false>{});
    else if (p.large) launch(LnShape<T, 128, 128, 2, 2, D, AD, BD, true>{});
    else if (!narrow) launch(LnShape<T, 64, 64, 2, 2, D, AD, BD, false>{});
    else launch(LnShape<T, 64, 64, 2, 2, D, AD, BD, true>{});
    TDGS_LAUNCHED();
    if (p.splits > 1) {
        k_linear_join<T><<<(unsigned)ceil_div((int64_t)r.P * (p.part_q / 8), kLnThreads), kLnThreads, 0, stream>>>(r);
        TDGS_LAUNCHED();
    }
    return TDGS_OK;
}

static int ln_check(const tdgs_linear* a) {
    TDGS_REQUIRE(a != nullptr, "linear: null arguments");
    TDGS_REQUIRE(known_dtype(a->dtype), "linear: unknown element type %d", a->dtype);
    TDGS_REQUIRE(a->activation >= TDGS_ACT_IDENTITY && a->activation <= TDGS_ACT_RELU, "linear: unknown activation %d",
                 a->activation);
    TDGS_REQUIRE(a->rows >= 0 && a->rows <= INT32_MAX - 65536, "linear: %lld rows", (long long)a->rows);
    TDGS_REQUIRE(a->in_features >= 1 && a->out_features >= 1 && a->in_features <= (1 << 20) && a->out_features <= (1 << 20) &&
                     (int64_t)a->in_features * a->out_features <= ((int64_t)1 << 36),
                 "linear: a weight matrix of %d x %d", a->in_features, a->out_features);
    TDGS_REQUIRE(a->weight_layout == TDGS_WEIGHT_IN_OUT || a->weight_layout == TDGS_WEIGHT_OUT_IN,
                 "linear: unknown weight layout %d", a->weight_layout);
    return TDGS_OK;
}

static int ln_check_rows(const tdgs_rows& v, const char* name, int32_t dtype, int64_t rows, int64_t cols, bool written) {
    TDGS_REQUIRE(v.data != nullptr, "linear: %s is null", name);
    TDGS_REQUIRE(aligned_to(v.data, (size_t)dtype_size(dtype)), "linear: %s is not aligned to its element type", name);
    TDGS_REQUIRE(v.stride >= 0, "linear: %s has a negative stride", name);
    if (written) TDGS_REQUIRE(rows <= 1 || v.stride >= cols, "linear: rows of %s overlap", name);
    return TDGS_OK;
}

static int ln_check_weight(const tdgs_rows& v, const char* name, const tdgs_linear* a, int32_t layout, bool written) {
    const bool in_out = layout == TDGS_WEIGHT_IN_OUT;
    return ln_check_rows(v, name, a->dtype, in_out ? a->in_features : a->out_features,
                         in_out ? a->out_features : a->in_features, written);
}

static LnMatrix ln_matrix(const tdgs_rows& v) { return {v.data, v.stride}; }

// The gradient's scratch: dz, its power of two, maxima and columns' sums, then a product's partial sums.
struct LnGradPlan {
    LnPlan dx, dw;
    int64_t dz_stride, per;
    int blocks;
    size_t dz, small, sums, part, bytes;
};

static LnGradPlan ln_grad_plan(const tdgs_linear* a) {
    LnGradPlan g;
    const bool slope = a->activation != TDGS_ACT_IDENTITY;
    g.dx = ln_plan(a->dtype, a->rows, a->in_features, a->out_features);
    // (the weight's gradient or its transpose, whichever is asked for: the larger of both is kept room for)
    g.dw = ln_plan(a->dtype, a->in_features, a->out_features, a->rows);
    const LnPlan t = ln_plan(a->dtype, a->out_features, a->in_features, a->rows);
    g.dz_stride = ceil_div(a->out_features, 8) * 8;
    g.dz = slope ? align_up((size_t)a->rows * g.dz_stride * dtype_size(a->dtype)) : 0;
    g.small = align_up((kLnTops + 1) * sizeof(float));
    const int64_t across = ceil_div(a->out_features, kWave * 8);
    int64_t blocks = ceil_div(2048, across);
    if (blocks > ceil_div(a->rows, 16)) blocks = ceil_div(a->rows, 16);
    g.per = ceil_div(a->rows, blocks > 0 ? blocks : 1);
    g.blocks = (int)(g.per > 0 ? ceil_div(a->rows, g.per) : 0);
    g.sums = align_up((size_t)g.blocks * a->out_features * sizeof(float));
    g.part = g.dx.bytes > g.dw.bytes ? g.dx.bytes : g.dw.bytes;
    if (t.bytes > g.part) g.part = t.bytes;
    g.bytes = g.dz + g.small + g.sums + g.part;
    return g;
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

size_t tdgs_linear_temp_bytes(const tdgs_linear* a, int32_t grad) {
    if (ln_check(a) != TDGS_OK) return 0;
    size_t bytes = ln_plan(a->dtype, a->rows, a->out_features, a->in_features).bytes;
    if (grad) {
        const size_t g = ln_grad_plan(a).bytes;
        if (g > bytes) bytes = g;
    }
    return bytes;
}

int tdgs_linear_forward(void* stream_, const tdgs_linear* a) {
    TDGS_TRY(ln_check(a));
    if (a->rows == 0) return TDGS_OK;
    TDGS_TRY(ln_check_rows(a->x, "x", a->dtype, a->rows, a->in_features, false));
    TDGS_TRY(ln_check_weight(a->weight, "the weight", a, a->weight_layout, false));
    TDGS_TRY(ln_check_rows(a->out, "out", a->dtype, a->rows, a->out_features, true));
    if (a->residual.data) TDGS_TRY(ln_check_rows(a->residual, "residual", a->dtype, a->rows, a->out_features, false));
    if (a->pre.data) TDGS_TRY(ln_check_rows(a->pre, "pre", a->dtype, a->rows, a->out_features, true));
    TDGS_REQUIRE(aligned_to(a->bias, (size_t)dtype_size(a->dtype)), "linear: bias is not aligned to its element type");
    const LnPlan p = ln_plan(a->dtype, a->rows, a->out_features, a->in_features);
    TDGS_REQUIRE(p.bytes == 0 || (a->temp && a->temp_bytes >= p.bytes && aligned_to(a->temp, 16)),
                 "linear: scratch of %zu bytes, %zu needed", a->temp ? a->temp_bytes : (size_t)0, p.bytes);
    LnArgs r = {};
    r.a = ln_matrix(a->x);
    r.b = ln_matrix(a->weight);
    r.P = (int32_t)a->rows;
    r.Q = a->out_features;
    r.R = a->in_features;
    r.act = a->activation;
    r.out = ln_matrix(a->out);
    r.residual = ln_matrix(a->residual);
    r.pre = ln_matrix(a->pre);
    r.bias = a->bias;
    hipStream_t stream = (hipStream_t)stream_;
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        return a->weight_layout == TDGS_WEIGHT_IN_OUT ? ln_product<T, true, false>(r, p, a->temp, stream)
                                                      : ln_product<T, true, true>(r, p, a->temp, stream);
    });
}

int tdgs_linear_grad(void* stream_, const tdgs_linear* a, const tdgs_linear_grads* g) {
    TDGS_TRY(ln_check(a));
    TDGS_REQUIRE(g != nullptr, "linear: null gradients");
    const bool slope = a->activation != TDGS_ACT_IDENTITY, rows = a->rows > 0;
    const bool want_dx = g->dx.data && rows, want_dw = g->dweight.data != nullptr, want_db = g->dbias != nullptr;
    if (!want_dx && !want_dw && !want_db) return TDGS_OK;
    if (rows) {
        TDGS_TRY(ln_check_rows(g->dout, "dout", a->dtype, a->rows, a->out_features, false));
        if (slope) TDGS_TRY(ln_check_rows(a->pre, "pre", a->dtype, a->rows, a->out_features, false));
    }
    if (want_dx) {
        TDGS_TRY(ln_check_weight(a->weight, "the weight", a, a->weight_layout, false));
        TDGS_TRY(ln_check_rows(g->dx, "dx", a->dtype, a->rows, a->in_features, true));
    }
    if (want_dw) {
        TDGS_REQUIRE(g->dweight_layout == TDGS_WEIGHT_IN_OUT || g->dweight_layout == TDGS_WEIGHT_OUT_IN,
                     "linear: unknown weight layout %d", g->dweight_layout);
        if (rows) TDGS_TRY(ln_check_rows(a->x, "x", a->dtype, a->rows, a->in_features, false));
        TDGS_TRY(ln_check_weight(g->dweight, "dweight", a, g->dweight_layout, true));
    }
    TDGS_REQUIRE(aligned_to(g->dbias, (size_t)dtype_size(a->dtype)), "linear: dbias is not aligned to its element type");
    LnGradPlan p = ln_grad_plan(a);
    TDGS_REQUIRE(!rows || (a->temp && a->temp_bytes >= p.bytes && aligned_to(a->temp, 16)),
                 "linear: scratch of %zu bytes, the gradient needs %zu", a->temp ? a->temp_bytes : (size_t)0, p.bytes);
    hipStream_t stream = (hipStream_t)stream_;
    const bool dw_in_out = g->dweight_layout == TDGS_WEIGHT_IN_OUT;
    if (!rows) {
        return with_dtype(a->dtype, [&](auto t) -> int {
            using T = decltype(t);
            const int64_t n = (int64_t)a->in_features * a->out_features;
            const int cols = dw_in_out ? a->out_features : a->in_features;
            if (want_dw)
                k_linear_zero<T><<<(unsigned)ceil_div(n, kLnThreads), kLnThreads, 0, stream>>>(
                    (T*)g->dweight.data, n / cols, cols, g->dweight.stride);
            if (want_db)
                k_linear_zero<T><<<(unsigned)ceil_div(a->out_features, kLnThreads), kLnThreads, 0, stream>>>(
                    (T*)g->dbias, 1, a->out_features, a->out_features);
            TDGS_LAUNCHED();
            return TDGS_OK;
        });
    }
    char* at = (char*)a->temp;
    LnGradArgs e = {};
    e.dout = ln_matrix(g->dout);
    e.pre = ln_matrix(a->pre);
    if (slope) e.dz = {at, p.dz_stride};
    at += p.dz;
    float* const top = (float*)at;
    at += p.small;
    e.sums = want_db ? (float*)at : nullptr;
    at += p.sums;
    void* const part = at;
    e.rows = a->rows;
    e.n = a->out_features;
    e.act = a->activation;
    e.blocks = p.blocks;
    e.per = p.per;
    // float16 and a slope: the products of both may pass the type's range, or leave it with few bits
    const bool ranged = slope && a->activation != TDGS_ACT_RELU && a->dtype == TDGS_F16;
    LnArgs r = {};
    r.a = slope ? e.dz : ln_matrix(g->dout);
    if (ranged) {
        e.top = top;
        e.tops = (int32_t)(a->rows < kLnTops ? a->rows : kLnTops);
        e.scale = top + kLnTops;
        r.scale = e.scale;
    }
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (ranged) {
            k_linear_top<T><<<(unsigned)e.tops, kLnThreads, 0, stream>>>(e, top);
            TDGS_LAUNCHED();
        }
        if (slope || want_db) {
            const dim3 grid((unsigned)ceil_div(a->out_features, kWave * 8), (unsigned)p.blocks);
            switch (a->activation) {
                case TDGS_ACT_IDENTITY: k_linear_dz<T, TDGS_ACT_IDENTITY><<<grid, kLnThreads, 0, stream>>>(e); break;
                case TDGS_ACT_SILU: k_linear_dz<T, TDGS_ACT_SILU><<<grid, kLnThreads, 0, stream>>>(e); break;
                case TDGS_ACT_GELU: k_linear_dz<T, TDGS_ACT_GELU><<<grid, kLnThreads, 0, stream>>>(e); break;
                default: k_linear_dz<T, TDGS_ACT_RELU><<<grid, kLnThreads, 0, stream>>>(e); break;
            }
            TDGS_LAUNCHED();
        }
        if (want_db) {
            k_linear_dbias<T><<<(unsigned)ceil_div(a->out_features, kLnBiasCols), kLnThreads, 0, stream>>>(
                e.sums, p.blocks, a->out_features, (T*)g->dbias);
            TDGS_LAUNCHED();
        }
        if (want_dx) {
            LnArgs x = r;   // dx = dz W^T
            x.b = ln_matrix(a->weight);
            x.P = (int32_t)a->rows;
            x.Q = a->in_features;
            x.R = a->out_features;
            x.out = ln_matrix(g->dx);
            if (a->weight_layout == TDGS_WEIGHT_IN_OUT) TDGS_TRY((ln_product<T, true, true>(x, p.dx, part, stream)));
            else TDGS_TRY((ln_product<T, true, false>(x, p.dx, part, stream)));
        }
        if (want_dw) {
            LnArgs w = r;   // dW = x^T dz, or its transpose dz^T x
            w.R = (int32_t)a->rows;
            w.out = ln_matrix(g->dweight);
            w.P = dw_in_out ? a->in_features : a->out_features;
            w.Q = dw_in_out ? a->out_features : a->in_features;
            w.b = dw_in_out ? r.a : ln_matrix(a->x);
            w.a = dw_in_out ? ln_matrix(a->x) : r.a;
            const LnPlan dw = ln_plan(a->dtype, w.P, w.Q, w.R);
            TDGS_TRY((ln_product<T, false, false>(w, dw, part, stream)));
        }
        return TDGS_OK;
    });
}

}  // extern "C"
