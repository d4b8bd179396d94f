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
// second kernel, which joins all that a call has left to join, in the order of the splits.
//
// The epilogue turns blocks through LDS, so that 16 bytes of a row are one lane's, and adds the bias, keeps z where
// wanted, applies the activation and adds the residual, all in 32 bits; only what is stored is rounded.
//
// What bounds the products: for 16-bit types the vector operations of the epilogue next to the matrix cores (32400 x 1024 ->
// 4096 bfloat16 with GELU, 314 to 340 us by card: matrix cores busy for 44%, vector issue for 65%; 8192^3 without an activation 870 us,
// 1260 TFLOP/s); for float the matrix cores (66 to 70% busy over 7503 x 387 x 1029, 79 us, of which some ten are the
// first tiles' way from memory and the last ones' back); for 34230 x 320 -> 320 memory (66 MB in 18 to 22 us); for few rows
// the call.
#include "internal.hpp"
#include "elem.hpp"
#include "activation.hpp"
#include "overlap.hpp"

namespace tdgs {

constexpr int kLnCus = 256;

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
    const float* scale;       // null, or out = *scale C, without a bias
    const void *a2, *b2;      // null, or C = A B + A2 B2 of matrices that lie as A and B do: the second half of the splits
};

// Elements of 16 bytes.
template <class T>
constexpr int ln_chunk() { return 16 / (int)sizeof(T); }
// Elements between LDS rows. Depth contiguous: 16 bytes of padding, and a read of 16 rows covers the banks once. Items
// contiguous: rows 16 banks apart for the transposing reads of four rows, four banks apart for single floats,
// whose two halves are eight rows apart.
template <class T, bool DEPTH, int N>
constexpr int ln_pitch() { return N + (DEPTH || sizeof(T) == 4 ? ln_chunk<T>() : 32); }

// A tile of MAJ memory rows x MIN elements on its way to LDS, by TH threads: a thread takes 16 bytes of every kStep-th
// row, loaded from a uniform base and an offset of its own, so that a step of the depth moves the base alone.
template <class T, int MAJ, int MIN, int TH, int PITCH>
struct LnTile {
    static constexpr int C = ln_chunk<T>();
    static constexpr int kStep = TH / (MIN / C);       // rows apart
    static constexpr int kPer = MAJ / kStep;
    static_assert(TH % (MIN / C) == 0 && MAJ % kStep == 0, "whole rows of threads");
    typedef uint32_t U4 __attribute__((ext_vector_type(4)));
    typedef T Ca __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    U4 r[kPer];
    uint32_t offset[kPer];   // bytes, from 16 bytes before the tile
    __device__ __forceinline__ static int row(int k) { return (int)threadIdx.x / (MIN / C) + k * kStep; }
    __device__ __forceinline__ static int col() { return (int)threadIdx.x % (MIN / C) * C; }
    // Of the tile's rows `maj` > 0 and of their elements `min` > 0 exist; the memory row holds C elements or more, before the
    // tile or in it. Chunks across its end, or behind it, are its last 16 bytes.
    __device__ __forceinline__ void place(int64_t stride, int maj, int min) {
        const int x = col() + C <= min ? col() : min - C;
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            offset[k] = (uint32_t)((row(k) < maj ? row(k) : maj - 1) * (int)(stride * sizeof(T)) + (x + C) * (int)sizeof(T));
    }
    __device__ __forceinline__ void load(const T* tile) {
        const char* const base = (const char*)tile - 16;
#pragma unroll
        for (int k = 0; k < kPer; ++k) r[k] = __builtin_bit_cast(U4, *reinterpret_cast<const Ca*>(base + offset[k]));
    }
    // The same by single elements, for memory rows of fewer than C of them.
    __device__ __forceinline__ void load_narrow(const T* tile, int64_t stride, int maj, int min) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int y = row(k) < maj ? row(k) : maj - 1;
            T e[C];
#pragma unroll
            for (int i = 0; i < C; ++i) e[i] = col() + i < min ? tile[y * stride + col() + i] : (T)0.0f;
            r[k] = __builtin_bit_cast(U4, e);
        }
    }
    template <bool NARROW>
    __device__ __forceinline__ void store(T* lds, int maj, int min) {
        if (!NARROW && min < MIN) {   // chunks across the rows' end
            if (col() >= min) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) r[k] = (U4)0;
            } else if (col() + C > min) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) r[k] = shift_down(r[k], (C - min % C) * (int)sizeof(T) * 8);
            }
        }
        if (maj < MAJ) {
#pragma unroll
            for (int k = 0; k < kPer; ++k)
                if (row(k) >= maj) r[k] = (U4)0;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) *reinterpret_cast<U4*>(lds + row(k) * PITCH + col()) = r[k];
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

// GELU as relu(z) - |z| cdf(-|z|), the tail by the formula of act_value: no selections, and twelve operations
// next to the exponential and the reciprocal instead of fifteen.
__device__ __forceinline__ float ln_gelu(float z) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
    const float e = __builtin_amdgcn_exp2f(z * (-0.5f * kLog2e) * z);
    float a = __builtin_fmaf(0.5f * 1.061405429f, t, -0.5f * 1.453152027f);
    a = __builtin_fmaf(a, t, 0.5f * 1.421413741f);
    a = __builtin_fmaf(a, t, -0.5f * 0.284496736f);
    a = __builtin_fmaf(a, t, 0.5f * 0.254829592f);
    // (infinity has a tail of 0, and 0 of it; NaN is the tail's)
    return __builtin_fmaf(-__builtin_amdgcn_fmed3f(fabsf(z), 0.0f, 1e30f), a * t * e, fmaxf(z, 0.0f));
}

// Its derivative: with s = |z| pdf(z) - cdf(-|z|), 1 + s for positive z and -s otherwise.
__device__ __forceinline__ float ln_gelu_slope(float z) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
    const float e = __builtin_amdgcn_exp2f(z * (-0.5f * kLog2e) * z);
    float a = __builtin_fmaf(0.5f * 1.061405429f, t, -0.5f * 1.453152027f);
    a = __builtin_fmaf(a, t, 0.5f * 1.421413741f);
    a = __builtin_fmaf(a, t, -0.5f * 0.284496736f);
    a = __builtin_fmaf(a, t, 0.5f * 0.254829592f);
    const float s = e * __builtin_fmaf(__builtin_amdgcn_fmed3f(fabsf(z), 0.0f, 1e30f), 0.39894228040143268f, -(a * t));
    return z > 0.0f ? 1.0f + s : -s;
}

template <int ACT>
__device__ __forceinline__ void ln_act8(float (&v)[8]) {
    float none;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (ACT == TDGS_ACT_GELU) v[i] = ln_gelu(v[i]);
        else v[i] = act_value<ACT, false>(v[i], &none);
    }
}
__device__ __forceinline__ void ln_activate(int act, float (&v)[8]) {
    switch (act) {
        case TDGS_ACT_SILU: ln_act8<TDGS_ACT_SILU>(v); break;
        case TDGS_ACT_GELU: ln_act8<TDGS_ACT_GELU>(v); break;
        case TDGS_ACT_RELU: ln_act8<TDGS_ACT_RELU>(v); break;
        default: break;
    }
}

// The end of n (1 to 8) neighbouring results q.. of row p: bias holds those of the bias, or zeros, and `residual`, where not
// null, what has been loaded of the residual.
template <class T>
__device__ __forceinline__ void ln_finish(const LnArgs& a, float scale, const float (&bias)[8], int64_t p, int q, int n,
                                          float (&v)[8], const typename LnVec<T>::Va* residual = nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a.scale ? v[i] * scale : v[i] + bias[i];   // (never both)
    if (a.pre.p) LnVec<T>::store((T*)a.pre.p + p * a.pre.stride + q, n, v);
    ln_activate(a.act, v);
    if (residual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += (float)(*residual)[i];
    } else if (a.residual.p) {
        float r[8];
        LnVec<T>::load((const T*)a.residual.p + p * a.residual.stride + q, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    LnVec<T>::store((T*)a.out.p + p * a.out.stride + q, n, v);
}
template <class T>
__device__ __forceinline__ void ln_bias(const LnArgs& a, int q, int n, float (&bias)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = 0.0f;
    if (a.bias && n > 0) LnVec<T>::load((const T*)a.bias + q, n, bias);
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

// The end of a wavefront's blocks, which start at (p0, q0).
template <class S>
__device__ __forceinline__ void ln_end(const LnArgs& a, const f32x16 (&acc)[S::NP][S::NQ], float* mem, int p0, int q0, int split) {
    using T = typename S::T;
    const int lane = (int)__lane_id();
    // 32 rows at a time through the wavefront's own part of LDS
    float* const turn = mem + (int)threadIdx.x / kWave * 32 * S::kTurn;
    const float scale = a.scale ? *a.scale : 1.0f;
    constexpr int kPerRow = S::NQ * 4;          // lanes of a row, with eight results each
    constexpr int kRows = kWave / kPerRow;
    const int x = lane % kPerRow * 8, q = q0 + x, n = min(8, a.Q - q);
    float bias[8];
    ln_bias<T>(a, q, n, bias);
    // The residual of 32 rows is on its way while the rows before are worked on.
    constexpr int kAhead = 32 / kRows;
    typename LnVec<T>::Va rest[2][kAhead];
    const bool ahead = a.residual.p && !a.part && a.Q % 8 == 0;
    auto fetch = [&](int i) {
#pragma unroll
        for (int r = 0; r < kAhead; ++r) {
            const int p = min(p0 + i * 32 + r * kRows + lane / kPerRow, a.P - 1);
            rest[i & 1][r] = *reinterpret_cast<const typename LnVec<T>::Va*>((const T*)a.residual.p + p * a.residual.stride + (n > 0 ? q : 0));
        }
    };
    if (ahead) fetch(0);
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
        if (ahead && i + 1 < S::NP) fetch(i + 1);
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
            const int y = r0 + lane / kPerRow, p = p0 + i * 32 + y;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(turn + y * S::kTurn + x);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(turn + y * S::kTurn + x + 4);
            if (p >= a.P || n <= 0) continue;
            if (a.part) {
                f32x4* const o = reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.P + p) * a.part_q + q);
                o[0] = lo;
                o[1] = hi;
            } else {
                float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                if (ahead) ln_finish<T>(a, scale, bias, p, q, n, v, &rest[i & 1][r0 / kRows]);
                else ln_finish<T>(a, scale, bias, p, q, n, v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Which tile a workgroup takes. Items that follow each other run on one XCD (xcd_band_item) at the same time, and go down
// kLnGroup tiles of rows before they go on to the next columns, so that fewer different pieces of A and B pass
// through its L2 together (8192^3 bfloat16 by 256x256 876 us, 920 row by row; by 128x256 980 and 1268).
constexpr int kLnGroup = 8;
struct LnPlace {
    int split, p, q;
    __device__ __forceinline__ explicit LnPlace(const LnArgs& a) {
        const int item = xcd_band_item(blockIdx.x, gridDim.x), tiles = a.tiles_p * a.tiles_q;
        split = item / tiles;
        const int tile = item - split * tiles, first = tile / (kLnGroup * a.tiles_q) * kLnGroup;
        const int rows = min(kLnGroup, a.tiles_p - first), rest = tile - first * a.tiles_q;
        q = rest / rows;
        p = first + rest - q * rows;
    }
};

// Two stages: while a step is multiplied, the next one's tiles are stored to LDS and the loads of the one after are in flight.
// float by 128x128, three workgroups a CU, or 64x64, eight: forward 8192 x 4096 x 4096 2222 us (124 TFLOP/s; a library product
// 1822) and 2327, 32400 x 512 x 2048 588 and 624, its weight's gradient 569 and 776; 7503 x 387 x 1029 97 (CUs idle) and
// 66 (a library product 61), 64800 x 64 x 512 63 and 56. Of 135 products, forward and weights' gradients, that were timed by
// both, ln_plan takes the faster one, or one within 2% of it, in 125, and loses 26% at most (64x64 always: 36%).
template <class S>
__global__ __launch_bounds__(S::TH) void k_linear(LnArgs a) {
    using T = typename S::T;
    __shared__ __attribute__((aligned(16))) char s_mem[S::kLds];
    T* const s = reinterpret_cast<T*>(s_mem);
    const int wave = (int)threadIdx.x / kWave, lane = (int)__lane_id();
    const int wp = wave / S::WQ * (S::BP / S::WP), wq = wave % S::WQ * (S::BQ / S::WQ);
    const LnPlace at(a);
    const int split = at.split, p0 = at.p * S::BP, q0 = at.q * S::BQ;
    const bool second = a.a2 && split >= a.splits / 2;
    const int r_begin = (second ? split - a.splits / 2 : split) * a.steps * S::BK, r_end = min(a.R, r_begin + a.steps * S::BK);
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
    const int64_t step_a = S::AD ? S::BK : S::BK * a.a.stride, step_b = S::BD ? S::BK : S::BK * a.b.stride;
    const T* pa = (const T*)(second ? a.a2 : a.a.p) + (S::AD ? p0 * a.a.stride + r_begin : r_begin * a.a.stride + p0);
    const T* pb = (const T*)(second ? a.b2 : a.b.p) + (S::BD ? q0 * a.b.stride + r_begin : r_begin * a.b.stride + q0);
    auto place = [&](int nr) {
        ta.place(a.a.stride, S::AD ? np : nr, S::AD ? nr : np);
        tb.place(a.b.stride, S::BD ? nq : nr, S::BD ? nr : nq);
    };
    // (in the order of the steps)
    auto load = [&](int step) {
        const int nr = r_end - r_begin - step * S::BK;
        if constexpr (S::NARROW) {
            ta.load_narrow(pa, a.a.stride, S::AD ? np : nr, S::AD ? nr : np);
            tb.load_narrow(pb, a.b.stride, S::BD ? nq : nr, S::BD ? nr : nq);
        } else {
            if (nr < S::BK) place(nr);
            ta.load(pa);
            tb.load(pb);
        }
        pa += step_a;
        pb += step_b;
    };
    auto store = [&](int step) {
        const int nr = r_end - r_begin - step * S::BK;
        T* const lds = s + (step & 1) * (S::kA + S::kB);
        ta.template store<S::NARROW>(lds, S::AD ? np : nr, S::AD ? nr : np);
        tb.template store<S::NARROW>(lds + S::kA, S::BD ? nq : nr, S::BD ? nr : nq);
    };
    if constexpr (!S::NARROW) place(S::BK);
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

    ln_end<S>(a, acc, reinterpret_cast<float*>(s_mem), p0 + wp, q0 + wq, split);
}

// ---- the same with tiles that go from memory to LDS directly ------------------------------------

// Rows of LDS are not padded then (a wavefront's 16 byte pieces arrive side by side); instead the pieces of a row change
// places by an exclusive or with bits of the row, so that a read covers the banks once: 16 neighbouring rows where
// the depth is contiguous, four rows x 64 bytes where the items are.
template <bool DEPTH, int MIN>
__device__ __forceinline__ int lf_key(int row) {
    if constexpr (!DEPTH) return MIN == 64 ? (row & 2) << 1 : (row & 3) << 2;
    else if constexpr (MIN == 32) return (row >> 2) & 3;
    else return (row >> 1) & 7;
}

template <class T, bool DEPTH, int MAJ, int MIN, int TH>
struct LfTile {
    static constexpr int CR = MIN / 8;             // pieces of a row
    static constexpr int kStep = TH / CR, kPer = MAJ / kStep;
    static_assert(sizeof(T) == 2 && TH % CR == 0 && MAJ % kStep == 0, "whole rows of threads");
    uint32_t offset[kPer];
    __device__ __forceinline__ static int row(int k) { return (int)threadIdx.x / CR + k * kStep; }
    __device__ __forceinline__ static int col(int k) { return (((int)threadIdx.x % CR) ^ lf_key<DEPTH, MIN>(row(k))) * 8; }
    __device__ __forceinline__ void place(int64_t stride, int maj, int min) {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            offset[k] = (uint32_t)((row(k) < maj ? row(k) : maj - 1) * (int)(stride * 2) + (col(k) < min ? col(k) : min - 8) * 2);
    }
    // All of the tile to LDS, in flight.
    __device__ __forceinline__ void start(const T* tile, uint32_t lds) const {
        const uint32_t at = __builtin_amdgcn_readfirstlane(lds + (uint32_t)threadIdx.x / kWave * 1024);
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                         :: "s"(at + k * TH * 16), "v"(offset[k]), "s"(tile) : "memory", "m0");
    }
    // A tile whose depth ends in it, through registers.
    __device__ __forceinline__ void tail(const T* tile, int64_t stride, T* lds, int maj, int min) const {
        typedef T V8u __attribute__((ext_vector_type(8), aligned(16)));
        typename Elem<T>::V8 r[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int y = row(k) < maj ? row(k) : maj - 1;
            const T* const p = tile + y * stride + col(k);
            if (col(k) + 8 <= min || !DEPTH) {
                r[k] = *reinterpret_cast<const V8u*>(tile + y * stride + (DEPTH || col(k) < min ? col(k) : min - 8));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) r[k][i] = col(k) + i < min ? p[i] : (T)0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (!DEPTH && row(k) >= maj) r[k] = zero8<T>();
            *reinterpret_cast<typename Elem<T>::V8a*>(lds + (threadIdx.x + k * TH) * 8) = r[k];
        }
    }
};

// The operands (ln_operand) of such a tile: N blocks of 32 items by NC chunks of the depth. Which piece a lane reads depends on
// the chunk where the depth is contiguous and on the block where the items are; those places are made once, and all else
// is a constant offset. (Left to itself, the compiler makes them again in every step: 25 vector operations next to 8
// products.)
template <class T, bool DEPTH, int MIN, int N, int NC>
struct LfOperands {
    static constexpr int K = DEPTH ? NC : N;
    uint32_t at[K];
    __device__ __forceinline__ LfOperands(uint32_t lds, int base) {
        const int l = (int)__lane_id();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int e;
            if constexpr (DEPTH) {
                e = (base + (l & 31)) * MIN + ((k * 2 + (l >> 5)) ^ lf_key<true, MIN>(l & 31)) * 8;
            } else {
                const int row = (l >> 5) * 8 + ((l & 15) >> 2), piece = (base + k * 32) / 8 + ((l >> 4) & 1) * 2 + ((l & 3) >> 1);
                e = row * MIN + (piece ^ lf_key<false, MIN>((l >> 2) & 3)) * 8 + (l & 1) * 4;
            }
            at[k] = lds + (uint32_t)e * (uint32_t)sizeof(T);
            asm volatile("" : "+v"(at[k]));
        }
    }
    // The places in the stage that starts `stage` bytes on.
    __device__ __forceinline__ LfOperands(const LfOperands& first, uint32_t stage) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at[k] = first.at[k] + stage;
            asm volatile("" : "+v"(at[k]));
        }
    }
    // Block i, chunk c.
    __device__ __forceinline__ typename Elem<T>::V8 fetch(int i, int c) const {
        if constexpr (DEPTH) {
            typedef __attribute__((address_space(3))) const typename Elem<T>::V8a* lp;
            return *(lp)(uintptr_t)(at[c] + (uint32_t)(i * 32 * MIN * (int)sizeof(T)));
        } else {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4* lp;
            const uint32_t p = at[i] + (uint32_t)(c * 16 * MIN * (int)sizeof(T));
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)p);
            const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)(p + 4 * MIN * (int)sizeof(T)));
            return __builtin_bit_cast(typename Elem<T>::V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

template <class T_, int BP_, int BQ_, int WP_, int WQ_, int BK_, int STAGES_, int PER_CU_, bool AD_, bool BD_>
struct LfShape {
    typedef T_ T;
    static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, BK = BK_, STAGES = STAGES_, PER_CU = PER_CU_;
    static constexpr bool AD = AD_, BD = BD_;
    static constexpr int TH = WP * WQ * kWave;
    static constexpr int NP = BP / WP / 32, NQ = BQ / WQ / 32;
    static constexpr int AMAJ = AD ? BP : BK, AMIN = AD ? BK : BP;
    static constexpr int BMAJ = BD ? BQ : BK, BMIN = BD ? BK : BQ;
    static constexpr int kA = BP * BK, kB = BQ * BK;
    static constexpr int kTurn = BQ / WQ + 4;
    static constexpr size_t kStages = STAGES * (size_t)(kA + kB) * sizeof(T);
    static constexpr size_t kEnd = (size_t)WP * WQ * 32 * kTurn * sizeof(float);
    static constexpr size_t kLds = kStages > kEnd ? kStages : kEnd;
};

template <int N>
__device__ __forceinline__ void lf_wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
// All wavefronts have read what they read from LDS, and all loads waited for before are there.
__device__ __forceinline__ void lf_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// S::STAGES - 1 steps are in flight; a step waits for its own loads, then for all wavefronts, and the place that the step before
// read is loaded again. The loads are instructions without a register to write, which the compiler does not wait for by
// itself: the waits here count them. (By registers as k_linear does it, with the same tiles, 32400 x 1024 -> 4096 took 398 us
// instead of 352 by 256x128 and 485 instead of 303 by 256x256.)
template <class S>
__global__ __launch_bounds__(S::TH, S::PER_CU * S::TH / 256) void k_linear_direct(LnArgs a) {
    using T = typename S::T;
    __shared__ __attribute__((aligned(1024))) char s_mem[S::kLds];
    T* const s = reinterpret_cast<T*>(s_mem);
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_mem;
    const int wave = (int)threadIdx.x / kWave;
    const int wp = wave / S::WQ * (S::BP / S::WP), wq = wave % S::WQ * (S::BQ / S::WQ);
    const LnPlace place(a);
    const int split = place.split, p0 = place.p * S::BP, q0 = place.q * S::BQ;
    const bool second = a.a2 && split >= a.splits / 2;
    const int r_begin = (second ? split - a.splits / 2 : split) * a.steps * S::BK, r_end = min(a.R, r_begin + a.steps * S::BK);
    const int steps = (r_end - r_begin) / S::BK, rest = (r_end - r_begin) % S::BK;

    f32x16 acc[S::NP][S::NQ];
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
        for (int j = 0; j < S::NQ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    LfTile<T, S::AD, S::AMAJ, S::AMIN, S::TH> ta;
    LfTile<T, S::BD, S::BMAJ, S::BMIN, S::TH> tb;
    const int np = min(S::BP, a.P - p0), nq = min(S::BQ, a.Q - q0);
    const int64_t step_a = S::AD ? S::BK : S::BK * a.a.stride, step_b = S::BD ? S::BK : S::BK * a.b.stride;
    const T* pa = (const T*)(second ? a.a2 : a.a.p) + (S::AD ? p0 * a.a.stride + r_begin : r_begin * a.a.stride + p0);
    const T* pb = (const T*)(second ? a.b2 : a.b.p) + (S::BD ? q0 * a.b.stride + r_begin : r_begin * a.b.stride + q0);
    ta.place(a.a.stride, S::AD ? np : S::BK, S::AD ? S::BK : np);
    tb.place(a.b.stride, S::BD ? nq : S::BK, S::BD ? S::BK : nq);
    constexpr int kStage = S::kA + S::kB, kLoads = decltype(ta)::kPer + decltype(tb)::kPer;
    auto start = [&](int stage) {
        const uint32_t at = lds + stage * kStage * (int)sizeof(T);
        ta.start(pa, at);
        tb.start(pb, at + S::kA * (int)sizeof(T));
        pa += step_a;
        pb += step_b;
    };
    constexpr int NC = S::BK / 16;
    const LfOperands<T, S::AD, S::AMIN, S::NP, NC> oa(lds, wp);
    const LfOperands<T, S::BD, S::BMIN, S::NQ, NC> ob(lds + S::kA * (int)sizeof(T), wq);
    auto multiply = [&](int stage) {
        const decltype(oa) la(oa, stage * kStage * (int)sizeof(T));
        const decltype(ob) lb(ob, stage * kStage * (int)sizeof(T));
        typename Elem<T>::V8 fa[2][S::NP], fb[2][S::NQ];
        auto fetch = [&](int c) {
#pragma unroll
            for (int i = 0; i < S::NP; ++i) fa[c & 1][i] = la.fetch(i, c);
#pragma unroll
            for (int j = 0; j < S::NQ; ++j) fb[c & 1][j] = lb.fetch(j, c);
        };
        fetch(0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c + 1 < NC) fetch(c + 1);
#pragma unroll
            for (int i = 0; i < S::NP; ++i)
#pragma unroll
                for (int j = 0; j < S::NQ; ++j) acc[i][j] = mma(fb[c & 1][j], fa[c & 1][i], acc[i][j]);
        }
        // the reads of the next chunk go between the products of this one
        constexpr int kReads = S::NP * (S::AD ? 1 : 2) + S::NQ * (S::BD ? 1 : 2), kProducts = S::NP * S::NQ;
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
#pragma unroll
        for (int c = 0; c + 1 < NC; ++c) {
#pragma unroll
            for (int m = 0; m < kProducts; ++m) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if ((m + 1) * kReads / kProducts > m * kReads / kProducts)
                    __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kProducts - 1) / kProducts, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);
    };
#pragma unroll
    for (int n = 0; n < S::STAGES - 1; ++n)
        if (n < steps) start(n);
    int stage = 0, next = S::STAGES - 1;
    const int all = steps + (rest > 0);
    for (int step = 0; step < all; ++step) {
        if (step + S::STAGES - 2 < steps) lf_wait_loads<(S::STAGES - 2) * kLoads>();
        else lf_wait_loads<0>();
        lf_barrier();
        if (step + S::STAGES - 1 < steps) start(next);
        if (step == steps) {   // the depth's end
            ta.tail(pa, a.a.stride, s + stage * kStage, S::AD ? np : rest, S::AD ? rest : np);
            tb.tail(pb, a.b.stride, s + stage * kStage + S::kA, S::BD ? nq : rest, S::BD ? rest : nq);
            lf_barrier();
        }
        multiply(stage);
        stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        next = next + 1 == S::STAGES ? 0 : next + 1;
    }
    lf_barrier();
    ln_end<S>(a, acc, reinterpret_cast<float*>(s_mem), p0 + wp, q0 + wq, split);
}

// Joins the splits' sums, eight neighbouring results by G threads, each of which takes every G-th split. Workgroup `block`.
constexpr int kLnThreads = 256;
template <class T, int G>
__device__ __forceinline__ void ln_join(const LnArgs& a, int block, f32x8* s) {
    constexpr int N = kLnThreads / G;
    const int chunks = a.part_q / 8, x = (int)threadIdx.x % N, y = (int)threadIdx.x / N;
    const int64_t i = (int64_t)block * N + x, all = (int64_t)a.P * chunks;
    const int64_t p = (i < all ? i : all - 1) / chunks;
    const int q = (int)((i < all ? i : all - 1) - p * chunks) * 8;
    f32x8 sum = {};
    for (int k = y; k < a.splits; k += G) sum += *reinterpret_cast<const f32x8*>(a.part + ((int64_t)k * a.P + p) * a.part_q + q);
    if constexpr (G > 1) {
        s[threadIdx.x] = sum;
        __syncthreads();
        if (y != 0) return;
#pragma unroll 4
        for (int g = 1; g < G; ++g) sum += s[g * N + x];
    }
    if (i >= all) return;
    float v[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sum[e];
    const int n = min(8, a.Q - q);
    ln_bias<T>(a, q, n, bias);
    ln_finish<T>(a, a.scale ? *a.scale : 1.0f, bias, p, q, n, v);
}

// dbias from the runs' sums: eight columns per workgroup.
constexpr int kLnBiasCols = 8;
template <class T>
__device__ __forceinline__ void ln_dbias(const float* __restrict__ sums, int blocks, int n, T* dbias, int block, float* s) {
    const int x = (int)threadIdx.x % kLnBiasCols, y = (int)threadIdx.x / kLnBiasCols, c = block * kLnBiasCols + x;
    float v = 0.0f;
    if (c < n) {
#pragma unroll 8
        for (int b = y; b < blocks; b += kLnThreads / kLnBiasCols) v += sums[(int64_t)b * n + c];
    }
    s[y * (kLnBiasCols + 1) + x] = v;
    for (int w = kLnThreads / kLnBiasCols / 2; w > 0; w >>= 1) {   // by halves, as k_linear_dz
        __syncthreads();
        if (y < w) s[y * (kLnBiasCols + 1) + x] += s[(y + w) * (kLnBiasCols + 1) + x];
    }
    if (y == 0 && c < n) dbias[c] = (T)s[x];
}

// What a call has to join, in one launch at its end: up to two products, and dbias.
struct LnJoins {
    LnArgs product[2];
    int32_t together[2], blocks[2];   // ln_join's G; workgroups
    int32_t products, sum_blocks, n, bias_blocks;
    const float* sums;
    void* dbias;
    int64_t grid() const {
        int64_t g = bias_blocks;
        for (int i = 0; i < products; ++i) g += blocks[i];
        return g;
    }
};
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_join(LnJoins j) {
    __shared__ f32x8 s[kLnThreads];
    int block = blockIdx.x;
    for (int i = 0; i < j.products; ++i) {
        if (block < j.blocks[i]) {
            switch (j.together[i]) {
                case 1: ln_join<T, 1>(j.product[i], block, s); return;
                case 4: ln_join<T, 4>(j.product[i], block, s); return;
                default: ln_join<T, 32>(j.product[i], block, s); return;
            }
        }
        block -= j.blocks[i];
    }
    ln_dbias<T>(j.sums, j.sum_blocks, j.n, (T*)j.dbias, block, (float*)s);
}

// ---- few rows: the weight is read once, by vectors, in one launch ----------------------------

// Up to eight rows (four of 16-bit types) fill a fraction of a tile of the matrix cores, and what counts is how soon and how fast the weight comes
// from memory: every thread loads 16 bytes of it at a time, several in flight, and multiplies them by the rows' elements in
// 32 bits. The depth is shared out over a workgroup's threads and joined by exchanges and in LDS.
constexpr int kLsThreads = 512, kLsRows = 8;

template <class T>
struct LsChunk {   // 16 bytes
    static constexpr int C = ln_chunk<T>();
    typedef T Va __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    float f[C];
    __device__ __forceinline__ void load(const T* p, int n) {   // n of them exist
        if (n >= C) {
            const Va v = *reinterpret_cast<const Va*>(p);
#pragma unroll
            for (int i = 0; i < C; ++i) f[i] = (float)v[i];
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i) f[i] = i < n ? (float)p[i] : 0.0f;
        }
    }
};

// Items contiguous: a workgroup takes four chunks of columns, whose lanes are neighbours, and a thread every 128th depth.
template <class T, int ROWS>
__global__ __launch_bounds__(kLsThreads) void k_linear_few_items(LnArgs a) {
    constexpr int C = ln_chunk<T>(), W = kLsThreads / kWave, U = 4;
    __shared__ float s[W][4][ROWS * C];
    const int t = (int)threadIdx.x, chunk = t & 3, q = ((int)blockIdx.x * 4 + chunk) * C, n = a.Q - q;
    float sum[ROWS][C] = {};
    if (n > 0) {
        const T* const b = (const T*)a.b.p + q;
        const T* const x = (const T*)a.a.p;
        for (int r0 = t >> 2; r0 < a.R; r0 += U * (kLsThreads / 4)) {
            LsChunk<T> w[U];
            float e[U][ROWS];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * (kLsThreads / 4), at = r < a.R ? r : a.R - 1;
                w[u].load(b + at * a.b.stride, n);
#pragma unroll
                for (int p = 0; p < ROWS; ++p) {
                    const int64_t i = (p < a.P ? p : 0) * a.a.stride + at;
                    e[u][p] = (float)x[i];
                    if (a.a2) e[u][p] += (float)((const T*)a.a2)[i];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r0 + u * (kLsThreads / 4) >= a.R) break;
#pragma unroll
                for (int p = 0; p < ROWS; ++p)
#pragma unroll
                    for (int i = 0; i < C; ++i) sum[p][i] = __builtin_fmaf(e[u][p], w[u].f[i], sum[p][i]);
            }
        }
    }
#pragma unroll
    for (int p = 0; p < ROWS; ++p)
#pragma unroll
        for (int i = 0; i < C; ++i) {
            float v = sum[p][i];
            for (int m = kWave / 2; m >= 4; m >>= 1) v += __shfl_xor(v, m, kWave);
            if (__lane_id() < 4) s[t / kWave][chunk][p * C + i] = v;
        }
    __syncthreads();
    // eight results to a thread
    constexpr int N = 4 * C / 8;
    for (int i = t; i < N * ROWS; i += kLsThreads) {
        const int p = i / N, c = i % N * 8, col = (int)blockIdx.x * 4 * C + c;
        if (p >= a.P || col >= a.Q) continue;
        float v[8], bias[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = 0.0f;
            for (int w = 0; w < W; ++w) v[k] += s[w][(c + k) / C][p * C + (c + k) % C];
        }
        const int left = min(8, a.Q - col);
        ln_bias<T>(a, col, left, bias);
        ln_finish<T>(a, a.scale ? *a.scale : 1.0f, bias, p, col, left, v);
    }
}

// Depth contiguous: a wavefront takes two columns, and a lane every 64th chunk of them.
template <class T, int ROWS>
__global__ __launch_bounds__(kLsThreads) void k_linear_few_depth(LnArgs a) {
    constexpr int C = ln_chunk<T>(), W = kLsThreads / kWave, COLS = 2, U = 2;
    __shared__ float s[W * COLS][ROWS];
    const int t = (int)threadIdx.x, lane = (int)__lane_id(), q0 = ((int)blockIdx.x * W + t / kWave) * COLS;
    float sum[COLS][ROWS] = {};
    for (int r0 = lane * C; r0 < a.R; r0 += U * kWave * C) {
        LsChunk<T> w[U][COLS], x[U][ROWS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * kWave * C, left = a.R - r, at = left > 0 ? r : 0;
#pragma unroll
            for (int c = 0; c < COLS; ++c) w[u][c].load((const T*)a.b.p + (q0 + c < a.Q ? q0 + c : a.Q - 1) * a.b.stride + at, left);
#pragma unroll
            for (int p = 0; p < ROWS; ++p) {
                const int64_t i = (p < a.P ? p : 0) * a.a.stride + at;
                x[u][p].load((const T*)a.a.p + i, left);
                if (a.a2) {
                    LsChunk<T> rest;
                    rest.load((const T*)a.a2 + i, left);
#pragma unroll
                    for (int c = 0; c < C; ++c) x[u][p].f[c] += rest.f[c];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int p = 0; p < ROWS; ++p)
#pragma unroll
                    for (int i = 0; i < C; ++i) sum[c][p] = __builtin_fmaf(x[u][p].f[i], w[u][c].f[i], sum[c][p]);
    }
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int p = 0; p < ROWS; ++p) {
            float v = sum[c][p];
            for (int m = kWave / 2; m > 0; m >>= 1) v += __shfl_xor(v, m, kWave);
            if (lane == 0) s[t / kWave * COLS + c][p] = v;
        }
    __syncthreads();
    constexpr int N = W * COLS / 8;
    for (int i = t; i < N * ROWS; i += kLsThreads) {
        const int p = i / N, c = i % N * 8, col = (int)blockIdx.x * W * COLS + c;
        if (p >= a.P || col >= a.Q) continue;
        float v[8], bias[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = s[c + k][p];
        const int left = min(8, a.Q - col);
        ln_bias<T>(a, col, left, bias);
        ln_finish<T>(a, a.scale ? *a.scale : 1.0f, bias, p, col, left, v);
    }
}

// ---- the gradient's elementwise part: dz = dout act'(z), and its columns' sums ------------------

struct LnGradArgs {
    LnMatrix dout, pre, dz;     // dz null: not wanted
    void* rest;                 // null, or what its rounding leaves of dz, which lies as dz does
    int64_t rows;
    int32_t n, act, blocks, shift;
    float* sums;                // blocks x n; null: not wanted
    void* dbias;                // with one block: they are dbias
    const float* top;           // float16: partial maxima of |dout|; null: dz is not scaled
    int32_t tops;
    float* scale;               // what undoes dz's power of two
};

// The largest |dout| of each workgroup's share (float16), which together go through memory from front to back.
constexpr int kLnTops = 1024;
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_top(LnGradArgs a, float* top) {
    __shared__ float s[kLnThreads / kWave];
    const int t = (int)threadIdx.x, across = 1 << a.shift, down = kLnThreads >> a.shift;
    float m = 0.0f;
    constexpr int U = 4;
    for (int q = (t & (across - 1)) * 8; q < a.n; q += across * 8) {
        for (int64_t r = (int64_t)blockIdx.x * U * down + (t >> a.shift); r < a.rows; r += (int64_t)gridDim.x * U * down) {
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u)
                LnVec<T>::load((const T*)a.dout.p + min(r + u * down, a.rows - 1) * a.dout.stride + q, min(8, a.n - q), v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[u][i]));
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

// Workgroup (x, y): 2^shift chunks of eight columns by 256 >> shift rows at a time, the workgroups' rows in turn: all of
// them together go through memory from front to back (64800 x 2048 bfloat16 with GELU, 796 MB: 155 us, 5.1 TB/s; with a run of
// rows for each 203). With the sums of the columns, if wanted, before dz is rounded.
template <class T, int ACT>
__global__ __launch_bounds__(kLnThreads) void k_linear_dz(LnGradArgs a) {
    __shared__ float s[kLnThreads * 8];
    const int t = (int)threadIdx.x, across = 1 << a.shift, down = kLnThreads >> a.shift;
    const int q = ((int)blockIdx.x * across + (t & (across - 1))) * 8, y = t >> a.shift;
    float up = 1.0f;
    if (a.top) {
        float m = 0.0f;
        for (int i = t; i < a.tops; i += kLnThreads) m = fmaxf(m, a.top[i]);
        for (int w = kWave / 2; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, kWave));
        s[t] = m;
        __syncthreads();
        for (int w = 0; w < kLnThreads; w += kWave) m = fmaxf(m, s[w]);
        __syncthreads();
        up = ln_range(m);
        if (blockIdx.x == 0 && blockIdx.y == 0 && t == 0) *a.scale = 1.0f / up;
    }
    const int n = a.n - q;
    float sum[8] = {};
    if (n > 0) {
        auto rows = [&](int64_t r, auto count) {   // this row and, `down` rows apart, those after it
            constexpr int U = decltype(count)::value;
            float d[U][8], z[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                LnVec<T>::load((const T*)a.dout.p + (r + u * down) * a.dout.stride + q, n, d[u]);
                if constexpr (ACT != TDGS_ACT_IDENTITY) LnVec<T>::load((const T*)a.pre.p + (r + u * down) * a.pre.stride + q, n, z[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float slope = 1.0f;
                    if constexpr (ACT == TDGS_ACT_GELU) slope = ln_gelu_slope(z[u][i]);
                    else if constexpr (ACT != TDGS_ACT_IDENTITY) act_value<ACT, true>(z[u][i], &slope);
                    d[u][i] *= slope;
                    sum[i] += d[u][i];
                    if constexpr (std::is_same<T, f16>::value) d[u][i] *= up;
                }
                if (a.dz.p) LnVec<T>::store((T*)a.dz.p + (r + u * down) * a.dz.stride + q, n, d[u]);
                if constexpr (sizeof(T) == 2) {
                    if (a.rest) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float left = d[u][i] - (float)(T)d[u][i];
                            d[u][i] = fabsf(left) < INFINITY ? left : 0.0f;   // (infinity and NaN are in dz)
                        }
                        LnVec<T>::store((T*)a.rest + (r + u * down) * a.dz.stride + q, n, d[u]);
                    }
                }
            }
        };
        constexpr int U = 2;
        const int64_t step = (int64_t)gridDim.y * U * down;
        for (int64_t r = (int64_t)blockIdx.y * U * down + y; r < a.rows; r += step) {
            if (r + (U - 1) * down < a.rows) {
                rows(r, std::integral_constant<int, U>{});
            } else {
                for (int u = 0; u < U; ++u)
                    if (r + u * down < a.rows) rows(r + u * down, std::integral_constant<int, 1>{});
            }
        }
    }
    if (!a.sums) return;
    // The threads of a column by halves: one after the other, the 256 of a narrow layer left 2.5 to 3 times the error.
#pragma unroll
    for (int i = 0; i < 8; ++i) s[t * 8 + i] = sum[i];
    for (int w = down / 2; w > 0; w >>= 1) {
        __syncthreads();
        if (t < w * across) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[t * 8 + i] += s[(t + w * across) * 8 + i];
        }
    }
    __syncthreads();
    for (int c = t; c < across * 8; c += kLnThreads) {
        const int col = (int)blockIdx.x * across * 8 + c;
        if (col >= a.n) break;
        if (a.dbias) ((T*)a.dbias)[col] = (T)s[c];
        else a.sums[(int64_t)blockIdx.y * a.n + col] = s[c];
    }
}

// What is zero without rows (dweight and dbias).
template <class T>
__global__ __launch_bounds__(kLnThreads) void k_linear_zero(T* p, int64_t rows, int cols, int64_t stride) {
    for (int64_t i = (int64_t)blockIdx.x * kLnThreads + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * kLnThreads)
        p[i / cols * stride + i % cols] = (T)0.0f;
}

// ---- host ----------------------------------------------------------------------------------

// The forms of a product: tile, depth of a step, workgroups per CU, and what they take by measurement, in us: a
// workgroup's start and end, a step of one alone on its CU, and a step's share where the CU is full. 256x256 needs the fewest
// bytes from LDS per product (1.93 us a step are 1110 TFLOP/s), but fills a CU alone, so that nothing is multiplied
// while it ends; two workgroups of 128x256, with half the registers, end beside each other (64800 x 512 -> 2048 bfloat16 with
// GELU: 223 us, 247 by 256x256; at a depth of 1024 they are nearly even, at 8192^3 it is 919 and 870). Small tiles leave fewer
// CUs idle (34230 x 320 -> 320 float16 with a residual: 20 us by 128x64, 25 by 128x128, 43 by 256x256).
struct LnForm {
    int bp, bq, bk, per_cu;
    float ends, alone, full;
};
enum { kLnStaged64, kLnStaged128, kLnDirect64, kLnDirect128x64, kLnDirect128, kLnDirect128x256, kLnDirect256, kLnForms };
template <class T>
constexpr int ln_depth() { return sizeof(T) == 4 ? 16 : 32; }
constexpr LnForm kLnF32[2] = {{64, 64, ln_depth<float>(), 8, 3.0f, 0.5f, 0.3f}, {128, 128, ln_depth<float>(), 3, 5.0f, 1.3f, 1.12f}};
constexpr LnForm kLn16[kLnForms] = {{64, 64, ln_depth<bf16>(), 6, 3.0f, 0.5f, 0.25f}, {128, 128, ln_depth<bf16>(), 3, 5.0f, 0.8f, 0.42f},
                                    {64, 64, 64, 4, 3.0f, 0.46f, 0.206f},  {128, 64, 64, 3, 4.0f, 0.6f, 0.34f},
                                    {128, 128, 64, 2, 5.0f, 0.85f, 0.59f}, {128, 256, 32, 2, 3.0f, 0.8f, 0.62f}, {256, 256, 64, 1, 12.0f, 1.93f, 1.93f}};
constexpr int kLnLeastSteps = 4;   // of a split

// How a product is cut.
struct LnPlan {
    int form, tiles_p, tiles_q, splits, steps, part_q;
    size_t bytes;
};

// The form and the splits that take the least time: rounds of the workgroups of the fullest CU, and the join, which
// reads at 6 TB/s what the splits have left in the last-level cache, one after the other. A last round of float is counted by the
// workgroups that are in it (128x128 puts three on a CU: eight are two rounds and two thirds, not three); the figures of the
// 16-bit forms were fitted to rounds that count whole.
// `two`: a sum of two products, each by as many splits.
static LnPlan ln_plan(int32_t dtype, int64_t P, int64_t Q, int64_t R, bool direct, bool two) {
    if (P < 1 || Q < 1 || R < 1) return {};
    const bool f32 = dtype == TDGS_F32;
    const int chunk = f32 ? 4 : 8;
    const bool narrow = P < chunk || Q < chunk || R < chunk;
    const bool pieces = direct && !f32 && !narrow;
    const int first = pieces ? kLnDirect64 : kLnStaged64;
    const int last = narrow ? kLnStaged64 : pieces ? kLnDirect256 : kLnStaged128;
    LnPlan best = {};
    float least = INFINITY;
    for (int form = first; form <= last; ++form) {
        const LnForm& f = f32 ? kLnF32[form] : kLn16[form];
        const int64_t tiles = ceil_div(P, f.bp) * ceil_div(Q, f.bq), steps = ceil_div(R, f.bk);
        for (int fill = 0; fill <= f.per_cu; ++fill) {   // one split, or as many as put `fill` workgroups on each CU
            int64_t splits = fill ? (int64_t)fill * kLnCus / tiles : 1;
            if (splits > steps / kLnLeastSteps) splits = steps / kLnLeastSteps;
            if (splits < 1 || (fill && splits == 1)) {
                if (fill) continue;
                splits = 1;
            }
            const int64_t per = ceil_div(steps, splits);
            splits = ceil_div(steps, per);
            const int64_t on = ceil_div(tiles * splits, kLnCus), whole = on / f.per_cu, rest = on % f.per_cu;
            auto round = [&](int64_t together) {
                return f.ends + per * (f.full * together > f.alone ? f.full * together : f.alone);
            };
            float time = whole ? (float)whole * round(f.per_cu) : 0.0f;
            if (rest) time += round(whole && !f32 ? f.per_cu : rest);
            if (splits > 1) time += 3.0f + 0.012f * splits + (float)splits * P * Q * 4.0f / 6e6f;
            if (time < least) {
                least = time;
                best.form = form;
                best.tiles_p = (int)ceil_div(P, f.bp);
                best.tiles_q = (int)ceil_div(Q, f.bq);
                best.splits = (int)splits;
                best.steps = (int)per;
            }
        }
    }
    if (two) best.splits *= 2;
    best.part_q = (int)(ceil_div(Q, 8) * 8);
    best.bytes = best.splits > 1 ? align_up((size_t)best.splits * P * best.part_q * sizeof(float)) : 0;
    return best;
}

// Whether an operand's tiles can go to LDS directly: 16 byte pieces on their boundaries, whole where the items are contiguous.
static bool ln_aligned(const LnMatrix& m, bool depth, int64_t items) {
    return aligned_to(m.p, 16) && m.stride % 8 == 0 && m.stride < (1 << 21) && (depth || items % 8 == 0);
}

// Whether a product of few rows goes by vectors. float: 1 to 8 rows x 4096 x 4096 take 22 to 28 us so, 30 by tiles; 512 x 2048
// 10 and 13 (9.5 of them the call). 16-bit types have tiles that are read faster than this: 1 and 4 rows x 2048 x 512 11
// and 13 us, 15 and 13 by tiles; but 8 rows 18 and 14, one row x 4096 x 4096 20 and 14. Where the items are contiguous, a thread
// takes its depths 512 at a time one after the other, and few columns make few workgroups: tiles split the depth then.
static bool ln_few(int64_t size, bool depth, int64_t P, int64_t Q, int64_t R) {
    if (!depth && R > 2048 && (size == 2 || Q < 1024)) return false;
    return size == 4 ? P <= kLsRows : P <= 4 && Q * R <= (1 << 21);
}

template <class T>
static int ln_launch_joins(const LnJoins& j, hipStream_t stream) {
    if (j.grid() == 0) return TDGS_OK;
    TDGS_REQUIRE(j.grid() <= INT32_MAX, "linear: too many results to join");
    k_linear_join<T><<<(unsigned)j.grid(), kLnThreads, 0, stream>>>(j);
    TDGS_LAUNCHED();
    return TDGS_OK;
}

// C = A B, with what follows it in `r`, but for the joining of splits, which is left to `joins`. Partial sums go to *temp, which is
// moved on behind them.
template <class T, bool AD, bool BD>
static int ln_product(LnArgs r, char** temp, LnJoins* joins, hipStream_t stream) {
    const int32_t dtype = sizeof(T) == 4 ? TDGS_F32 : std::is_same<T, bf16>::value ? TDGS_BF16 : TDGS_F16;
    if (AD && ln_few(sizeof(T), BD, r.P, r.Q, r.R)) {
        auto few = [&](auto rows) {
            constexpr int ROWS = decltype(rows)::value;
            const int64_t cols = BD ? kLsThreads / kWave * 2 : 4 * ln_chunk<T>();
            if constexpr (BD) k_linear_few_depth<T, ROWS><<<(unsigned)ceil_div(r.Q, cols), kLsThreads, 0, stream>>>(r);
            else k_linear_few_items<T, ROWS><<<(unsigned)ceil_div(r.Q, cols), kLsThreads, 0, stream>>>(r);
        };
        if (r.P == 1) few(std::integral_constant<int, 1>{});
        else if (r.P <= 4) few(std::integral_constant<int, 4>{});
        else if constexpr (sizeof(T) == 4) few(std::integral_constant<int, kLsRows>{});
        TDGS_LAUNCHED();
        return TDGS_OK;
    }
    const bool aligned = sizeof(T) == 2 && ln_aligned(r.a, AD, r.P) && ln_aligned(r.b, BD, r.Q);
    const LnPlan p = ln_plan(dtype, r.P, r.Q, r.R, aligned, r.a2 != nullptr);
    r.tiles_p = p.tiles_p;
    r.tiles_q = p.tiles_q;
    r.splits = p.splits;
    r.steps = p.steps;
    r.part_q = p.part_q;
    r.part = p.splits > 1 ? (float*)*temp : nullptr;
    *temp += p.bytes;
    const int64_t grid = (int64_t)p.tiles_p * p.tiles_q * p.splits;
    // (a launch has fewer than 2^32 threads)
    TDGS_REQUIRE(grid * (p.form == kLnDirect128x256 || p.form == kLnDirect256 ? 512 : 256) <= UINT32_MAX,
                 "linear: %lld x %lld results are too many tiles for one call", (long long)r.P, (long long)r.Q);
    constexpr int C = ln_chunk<T>(), D = ln_depth<T>();
    auto staged = [&](auto shape) {
        using S = decltype(shape);
        k_linear<S><<<(unsigned)grid, S::TH, 0, stream>>>(r);
    };
    auto direct = [&](auto shape) {
        using S = decltype(shape);
        k_linear_direct<S><<<(unsigned)grid, S::TH, 0, stream>>>(r);
    };
    if ((AD ? r.R : r.P) < C || (BD ? r.R : r.Q) < C) {   // (the plan of such a product has the smallest tiles)
        staged(LnShape<T, 64, 64, 2, 2, D, AD, BD, true>{});
    } else if (p.form == kLnStaged64) {
        staged(LnShape<T, 64, 64, 2, 2, D, AD, BD, false>{});
    } else if (p.form == kLnStaged128) {
        staged(LnShape<T, 128, 128, 2, 2, D, AD, BD, false>{});
    } else if constexpr (sizeof(T) == 2) {
        if (p.form == kLnDirect64) direct(LfShape<T, 64, 64, 2, 2, 64, 2, 4, AD, BD>{});
        else if (p.form == kLnDirect128x64) direct(LfShape<T, 128, 64, 2, 2, 64, 2, 3, AD, BD>{});
        else if (p.form == kLnDirect128) direct(LfShape<T, 128, 128, 2, 2, 64, 2, 2, AD, BD>{});
        else if (p.form == kLnDirect128x256) direct(LfShape<T, 128, 256, 2, 4, 32, 3, 2, AD, BD>{});
        else direct(LfShape<T, 256, 256, 2, 4, 64, 2, 1, AD, BD>{});
    }
    TDGS_LAUNCHED();
    if (p.splits > 1) {
        const int i = joins->products++, g = p.splits < 8 ? 1 : p.splits < 64 ? 4 : 32;
        joins->product[i] = r;
        joins->together[i] = g;
        const int64_t blocks = ceil_div((int64_t)r.P * (p.part_q / 8), kLnThreads / g);
        TDGS_REQUIRE(blocks <= INT32_MAX, "linear: too many results to join");
        joins->blocks[i] = (int32_t)blocks;
    }
    return TDGS_OK;
}

static int ln_check(const tdgs_linear* a) {
    TDGS_REQUIRE(a != nullptr, "linear: null arguments");
    TDGS_REQUIRE(known_dtype(a->dtype), "linear: unknown element type %d", a->dtype);
    TDGS_REQUIRE(a->activation >= TDGS_ACT_IDENTITY && a->activation <= TDGS_ACT_RELU, "linear: unknown activation %d",
                 a->activation);
    TDGS_REQUIRE(a->rows >= 0 && a->rows <= INT32_MAX - (1 << 20), "linear: %lld rows", (long long)a->rows);
    TDGS_REQUIRE(a->in_features >= 1 && a->out_features >= 1 && a->in_features <= (1 << 20) && a->out_features <= (1 << 20) &&
                     (int64_t)a->in_features * a->out_features <= ((int64_t)1 << 36),
                 "linear: a weight matrix of %d x %d", a->in_features, a->out_features);
    TDGS_REQUIRE(a->weight_layout == TDGS_WEIGHT_IN_OUT || a->weight_layout == TDGS_WEIGHT_OUT_IN,
                 "linear: unknown weight layout %d", a->weight_layout);
    return TDGS_OK;
}

// Tiles of up to 128 rows (256 of at most 2^22 bytes each where they go to LDS directly) are addressed by 32 bits.
constexpr int64_t kLnRowBytes = 1 << 24;

static int ln_check_rows(const tdgs_rows& v, const char* name, int32_t dtype, int64_t rows, int64_t cols, bool written) {
    TDGS_REQUIRE(v.data != nullptr, "linear: %s is null", name);
    TDGS_REQUIRE(aligned_to(v.data, (size_t)dtype_size(dtype)), "linear: %s is not aligned to its element type", name);
    TDGS_REQUIRE(v.stride >= 0, "linear: %s has a negative stride", name);
    if (written) TDGS_REQUIRE(rows <= 1 || v.stride >= cols, "linear: rows of %s overlap", name);
    else TDGS_REQUIRE(rows <= 1 || v.stride * dtype_size(dtype) <= kLnRowBytes,
                      "linear: rows of %s are too far apart: %lld bytes, %lld at most", name,
                      (long long)(v.stride * dtype_size(dtype)), (long long)kLnRowBytes);
    return TDGS_OK;
}

static int ln_check_weight(const tdgs_rows& v, const char* name, const tdgs_linear* a, int32_t layout, bool written) {
    const bool in_out = layout == TDGS_WEIGHT_IN_OUT;
    return ln_check_rows(v, name, a->dtype, in_out ? a->in_features : a->out_features,
                         in_out ? a->out_features : a->in_features, written);
}

static LnMatrix ln_matrix(const tdgs_rows& v) { return {v.data, v.stride}; }
// An operand: the stride of a single row means nothing, and must not be calculated with.
static LnMatrix ln_operand_rows(const tdgs_rows& v, int64_t rows, int64_t cols) { return {v.data, rows > 1 ? v.stride : cols}; }

// What a matrix, or (layout) a weight matrix, or a vector covers.
static ByteRows ln_bytes(const tdgs_rows& v, const tdgs_linear* a, int64_t rows, int64_t cols) {
    const int64_t size = (int64_t)dtype_size(a->dtype);
    return ByteRows(v.data, v.data ? rows : 0, rows > 1 ? v.stride * size : 0, cols * size);
}
static ByteRows ln_weight_bytes(const tdgs_rows& v, const tdgs_linear* a, int32_t layout) {
    return layout == TDGS_WEIGHT_IN_OUT ? ln_bytes(v, a, a->in_features, a->out_features)
                                        : ln_bytes(v, a, a->out_features, a->in_features);
}
static ByteRows ln_vector_bytes(const void* v, const tdgs_linear* a) { return ln_bytes({(void*)v, 0}, a, 1, a->out_features); }

// Refuses `written` where it shares memory with one of the others: tiles of those are read, or written, at any time.
struct LnNamed {
    ByteRows rows;
    const char* name;
};
static int ln_check_apart(const LnNamed& written, std::initializer_list<LnNamed> others) {
    for (const LnNamed& o : others)
        TDGS_REQUIRE(!rows_overlap(written.rows, o.rows), "linear: %s overlaps %s", written.name, o.name);
    return TDGS_OK;
}

static LnMatrix ln_weight(const tdgs_linear* a) {
    return a->weight_layout == TDGS_WEIGHT_IN_OUT ? ln_operand_rows(a->weight, a->in_features, a->out_features)
                                                  : ln_operand_rows(a->weight, a->out_features, a->in_features);
}

// Up to so many elements of dz, which 16 bits round once more than the results, its products are taken of two operands, the second
// holding what the rounding leaves of the first: the errors of dx and dweight are 1.00 times those of the exact result rounded
// once instead of 1.40 to 1.42, for every size. What it costs decides: these calls are mostly latency (the whole gradient with
// GELU, one operand and two, in a graph: 256 x 256 -> 256 bfloat16 12 and 15 us, 64 x 1024 -> 1024 24 and 31, 128 x 2048 -> 512 13
// and 21, 32 x 1024 -> 2048 19 and 35), large ones would take both products' time again (64800 x 512 -> 2048: 293 of 468 us).
constexpr int64_t kLnFewSlopes = 1 << 16;

// The gradient's scratch: dz, its power of two, maxima and columns' sums, then a product's partial sums.
struct LnGradPlan {
    int64_t dz_stride;
    int blocks, shift;
    bool two;
    size_t dz, small, sums, part, bytes;
};

// Scratch of a product, whatever its operands' alignment.
static size_t ln_part_bytes(int32_t dtype, int64_t P, int64_t Q, int64_t R, bool two) {
    const size_t a = ln_plan(dtype, P, Q, R, false, two).bytes, b = ln_plan(dtype, P, Q, R, true, two).bytes;
    return a > b ? a : b;
}

static LnGradPlan ln_grad_plan(const tdgs_linear* a) {
    LnGradPlan g;
    const bool slope = a->activation != TDGS_ACT_IDENTITY;
    g.dz_stride = ceil_div(a->out_features, 8) * 8;
    g.two = slope && a->activation != TDGS_ACT_RELU && a->dtype != TDGS_F32 && a->rows * a->out_features <= kLnFewSlopes;
    g.dz = slope ? align_up((size_t)a->rows * g.dz_stride * dtype_size(a->dtype)) : 0;
    g.small = align_up((kLnTops + 1) * sizeof(float));
    g.shift = 0;
    while (g.shift < 6 && (8 << g.shift) < a->out_features) ++g.shift;
    const int64_t down = kLnThreads >> g.shift;
    int64_t blocks = ceil_div(1024, ceil_div(a->out_features, 8 << g.shift));
    // (a block of eight turns is as quick as the join of several)
    const int64_t turns = ceil_div(a->rows, 2 * down);
    if (blocks > turns) blocks = turns <= 8 ? 1 : turns;
    g.blocks = (int)blocks;
    g.sums = align_up((size_t)g.blocks * a->out_features * sizeof(float));
    // dx and (the weight's gradient or its transpose, whichever is asked for)
    const size_t dw = ln_part_bytes(a->dtype, a->in_features, a->out_features, a->rows, g.two);
    const size_t t = ln_part_bytes(a->dtype, a->out_features, a->in_features, a->rows, g.two);
    g.part = ln_part_bytes(a->dtype, a->rows, a->in_features, a->out_features, g.two) + (dw > t ? dw : t);
    g.bytes = (g.two ? 2 : 1) * g.dz + g.small + g.sums + g.part;
    return g;
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

size_t tdgs_linear_temp_bytes(const tdgs_linear* a, int32_t grad) {
    if (ln_check(a) != TDGS_OK) return 0;
    size_t bytes = ln_part_bytes(a->dtype, a->rows, a->out_features, a->in_features, false);
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
    // (tiles of x and of the weight are read while others of the results are written)
    TDGS_REQUIRE(a->out.data != a->x.data && a->out.data != a->weight.data, "linear: out is also an operand");
    TDGS_REQUIRE(!a->pre.data || (a->pre.data != a->out.data && a->pre.data != a->x.data && a->pre.data != a->weight.data &&
                                  a->pre.data != a->residual.data),
                 "linear: pre is also another tensor of the call");
    const size_t bytes = ln_part_bytes(a->dtype, a->rows, a->out_features, a->in_features, false);
    TDGS_REQUIRE(bytes == 0 || (a->temp && a->temp_bytes >= bytes && aligned_to(a->temp, 16)),
                 "linear: scratch of %zu bytes, %zu needed", a->temp ? a->temp_bytes : (size_t)0, bytes);
    const LnNamed x = {ln_bytes(a->x, a, a->rows, a->in_features), "x"}, w = {ln_weight_bytes(a->weight, a, a->weight_layout), "the weight"},
                  bias = {ln_vector_bytes(a->bias, a), "the bias"}, out = {ln_bytes(a->out, a, a->rows, a->out_features), "out"},
                  residual = {ln_bytes(a->residual, a, a->rows, a->out_features), "the residual"},
                  pre = {ln_bytes(a->pre, a, a->rows, a->out_features), "pre"};
    TDGS_TRY(ln_check_apart(out, {x, w, bias}));
    TDGS_REQUIRE(same_or_apart(out.rows, residual.rows), "linear: out overlaps the residual without being it");
    TDGS_TRY(ln_check_apart(pre, {x, w, bias, residual, out}));
    LnArgs r = {};
    r.a = ln_operand_rows(a->x, a->rows, a->in_features);
    r.b = ln_weight(a);
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
        LnJoins joins = {};
        char* at = (char*)a->temp;
        if (a->weight_layout == TDGS_WEIGHT_IN_OUT) TDGS_TRY((ln_product<T, true, false>(r, &at, &joins, stream)));
        else TDGS_TRY((ln_product<T, true, true>(r, &at, &joins, stream)));
        return ln_launch_joins<T>(joins, stream);
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
    if (rows) {   // (the products follow one another)
        TDGS_REQUIRE(!want_dx || (g->dx.data != g->dout.data && g->dx.data != a->weight.data && (!slope || g->dx.data != a->pre.data) &&
                                  (!want_dw || (g->dx.data != a->x.data && g->dx.data != g->dweight.data))),
                     "linear: dx is also another tensor of the call");
        TDGS_REQUIRE(!want_dw || (g->dweight.data != g->dout.data && g->dweight.data != a->x.data &&
                                  (!want_dx || g->dweight.data != a->weight.data) && (!slope || g->dweight.data != a->pre.data)),
                     "linear: dweight is also another tensor of the call");
    }
    LnGradPlan p = ln_grad_plan(a);
    TDGS_REQUIRE(!rows || (a->temp && a->temp_bytes >= p.bytes && aligned_to(a->temp, 16)),
                 "linear: scratch of %zu bytes, the gradient needs %zu", a->temp ? a->temp_bytes : (size_t)0, p.bytes);
    const bool dw_in_out = g->dweight_layout == TDGS_WEIGHT_IN_OUT;
    if (rows) {   // (of the operands those that are read)
        const tdgs_rows none = {};
        const LnNamed dout = {ln_bytes(g->dout, a, a->rows, a->out_features), "dout"},
                      pre = {ln_bytes(slope ? a->pre : none, a, a->rows, a->out_features), "pre"},
                      x = {ln_bytes(want_dw ? a->x : none, a, a->rows, a->in_features), "x"},
                      w = {ln_weight_bytes(want_dx ? a->weight : none, a, a->weight_layout), "the weight"},
                      dx = {ln_bytes(g->dx, a, a->rows, a->in_features), "dx"},
                      dw = {ln_weight_bytes(g->dweight, a, g->dweight_layout), "dweight"}, db = {ln_vector_bytes(g->dbias, a), "dbias"};
        TDGS_TRY(ln_check_apart(dx, {dout, pre, x, w, dw}));
        TDGS_TRY(ln_check_apart(dw, {dout, pre, x, w}));
        TDGS_TRY(ln_check_apart(db, {dout, pre, x, w, dx, dw}));
    }
    hipStream_t stream = (hipStream_t)stream_;
    if (!rows) {
        return with_dtype(a->dtype, [&](auto t) -> int {
            using T = decltype(t);
            const int64_t n = (int64_t)a->in_features * a->out_features;
            const int cols = dw_in_out ? a->out_features : a->in_features;
            if (want_dw)
                k_linear_zero<T><<<(unsigned)std::min<int64_t>(ceil_div(n, kLnThreads), 1 << 16), kLnThreads, 0, stream>>>(
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
    if (p.two) {
        e.rest = at;
        at += p.dz;
    }
    float* const top = (float*)at;
    at += p.small;
    e.sums = want_db ? (float*)at : nullptr;
    e.dbias = p.blocks == 1 ? g->dbias : nullptr;
    at += p.sums;
    e.rows = a->rows;
    e.n = a->out_features;
    e.act = a->activation;
    e.blocks = p.blocks;
    e.shift = p.shift;
    // float16 and a slope: the products of both may pass the type's range, or leave it with few bits
    const bool ranged = slope && a->activation != TDGS_ACT_RELU && a->dtype == TDGS_F16;
    LnArgs r = {};
    r.a = slope ? e.dz : ln_operand_rows(g->dout, a->rows, a->out_features);
    if (ranged) {
        e.top = top;
        const int64_t runs = ceil_div(a->rows, 4 * (kLnThreads >> p.shift));
        e.tops = (int32_t)(runs < kLnTops ? runs : kLnTops);
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
            const dim3 grid((unsigned)ceil_div(a->out_features, 8 << p.shift), (unsigned)p.blocks);
            switch (a->activation) {
                case TDGS_ACT_IDENTITY: k_linear_dz<T, TDGS_ACT_IDENTITY><<<grid, kLnThreads, 0, stream>>>(e); break;
                case TDGS_ACT_SILU: k_linear_dz<T, TDGS_ACT_SILU><<<grid, kLnThreads, 0, stream>>>(e); break;
                case TDGS_ACT_GELU: k_linear_dz<T, TDGS_ACT_GELU><<<grid, kLnThreads, 0, stream>>>(e); break;
                default: k_linear_dz<T, TDGS_ACT_RELU><<<grid, kLnThreads, 0, stream>>>(e); break;
            }
            TDGS_LAUNCHED();
        }
        LnJoins joins = {};
        if (want_db && !e.dbias) {
            joins.sums = e.sums;
            joins.sum_blocks = p.blocks;
            joins.n = a->out_features;
            joins.dbias = g->dbias;
            joins.bias_blocks = (int32_t)ceil_div(a->out_features, kLnBiasCols);
        }
        if (want_dx) {
            LnArgs x = r;   // dx = dz W^T
            x.b = ln_weight(a);
            x.a2 = e.rest;
            if (e.rest) x.b2 = x.b.p;
            x.P = (int32_t)a->rows;
            x.Q = a->in_features;
            x.R = a->out_features;
            x.out = ln_matrix(g->dx);
            if (a->weight_layout == TDGS_WEIGHT_IN_OUT) TDGS_TRY((ln_product<T, true, true>(x, &at, &joins, stream)));
            else TDGS_TRY((ln_product<T, true, false>(x, &at, &joins, stream)));
        }
        if (want_dw) {
            LnArgs w = r;   // dW = x^T dz, or its transpose dz^T x
            w.R = (int32_t)a->rows;
            w.out = ln_matrix(g->dweight);
            w.P = dw_in_out ? a->in_features : a->out_features;
            w.Q = dw_in_out ? a->out_features : a->in_features;
            const LnMatrix rows_x = ln_operand_rows(a->x, a->rows, a->in_features);
            w.b = dw_in_out ? r.a : rows_x;
            w.a = dw_in_out ? rows_x : r.a;
            if (e.rest) {
                w.a2 = dw_in_out ? rows_x.p : e.rest;
                w.b2 = dw_in_out ? e.rest : rows_x.p;
            }
            TDGS_TRY((ln_product<T, false, false>(w, &at, &joins, stream)));
        }
        return ln_launch_joins<T>(joins, stream);
    });
}

}  // extern "C"
