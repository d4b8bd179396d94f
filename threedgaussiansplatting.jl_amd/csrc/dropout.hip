// dropout.hip — dropout by a counter-based generator: the mask is a function of seed, call and element,
// computed where it is needed, forward and backward, and never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror & Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) encrypts
// the counter (element / 4, call) with the seed as key into the four words of four neighbouring elements. All 32
// bits decide, so that any p is met to 2^-32. Ten rounds for four elements are as much as the memory is for: 64800 x 1024
// bfloat16 with a residual take 69 us (398 MB, 5.8 TB/s, partly from the last-level cache) with vector issue busy for 92%.
#include "internal.hpp"
#include "elem.hpp"
#include "overlap.hpp"
#include "philox.hpp"

namespace tdgs {

constexpr int kDrThreads = 256;

struct DrArgs {
    const void *x, *residual;
    void* out;
    int64_t xs, rs, os;      // strides between rows
    int64_t rows, cols;
    PhiloxKey key;
    uint64_t call;
    const uint64_t* call_dev;
    DropRule rule;
    int32_t row_shift;       // 2^row_shift threads share a row
};

// A thread's VW neighbouring elements of a row; with VW > 1 they start on a multiple of four of the whole
// tensor, so that whole words of the generator are used. The threads of a workgroup stand side by side over
// 2^row_shift vectors of a row and 256 >> row_shift rows; contiguous tensors are one row.
template <class T, int VW>
__global__ __launch_bounds__(kDrThreads) void k_dropout(DrArgs a) {
    typedef T V __attribute__((ext_vector_type(VW)));
    typedef T Va __attribute__((ext_vector_type(VW), aligned(sizeof(T))));
    const uint64_t call = a.call_dev ? *a.call_dev : a.call;
    const int lane = (int)threadIdx.x & ((1 << a.row_shift) - 1), sub = (int)threadIdx.x >> a.row_shift;
    const int64_t vectors = (a.cols + VW - 1) / VW, step = (int64_t)gridDim.x << a.row_shift;
    const int64_t row_step = (int64_t)gridDim.y * (kDrThreads >> a.row_shift);
    for (int64_t row = (int64_t)blockIdx.y * (kDrThreads >> a.row_shift) + sub; row < a.rows; row += row_step) {
        const T* const x = (const T*)a.x + row * a.xs;
        const T* const r = a.residual ? (const T*)a.residual + row * a.rs : nullptr;
        T* const out = (T*)a.out + row * a.os;
        for (int64_t v = ((int64_t)blockIdx.x << a.row_shift) + lane; v < vectors; v += step) {
            const int64_t c = v * VW;
            const uint64_t e = (uint64_t)(row * a.cols + c);
            if constexpr (VW == 1) {
                const bool keep = a.rule.keeps(philox(a.key, e >> 2, call).w[e & 3]);
                const float y = keep ? (float)x[c] * a.rule.scale : 0.0f;
                out[c] = (T)(r ? (float)r[c] + y : y);
            } else {
                const int n = (int)(a.cols - c < VW ? a.cols - c : VW);
                V vx, vr;
                if (n == VW) {
                    vx = *reinterpret_cast<const Va*>(x + c);
                    if (r) vr = *reinterpret_cast<const Va*>(r + c);
                } else {
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        vx[i] = i < n ? x[c + i] : (T)0.0f;
                        if (r) vr[i] = i < n ? r[c + i] : (T)0.0f;
                    }
                }
                V vo;
#pragma unroll
                for (int g = 0; g < VW / 4; ++g) {
                    const Philox4 w = philox(a.key, (e >> 2) + g, call);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y = a.rule.keeps(w.w[i]) ? (float)vx[4 * g + i] * a.rule.scale : 0.0f;
                        vo[4 * g + i] = (T)(r ? (float)vr[4 * g + i] + y : y);
                    }
                }
                if (n == VW) {
                    *reinterpret_cast<Va*>(out + c) = vo;
                } else {
#pragma unroll
                    for (int i = 0; i < VW; ++i)
                        if (i < n) out[c + i] = vo[i];
                }
            }
        }
    }
}

static int dr_check_rows(const tdgs_rows* v, const char* name, const tdgs_dropout* a, bool written) {
    TDGS_REQUIRE(v->data != nullptr, "dropout: %s is null", name);
    TDGS_REQUIRE(aligned_to(v->data, (size_t)dtype_size(a->dtype)), "dropout: %s is not aligned to its element type", name);
    TDGS_REQUIRE(v->stride >= 0, "dropout: %s has a negative stride", name);
    if (written) TDGS_REQUIRE(a->rows <= 1 || v->stride >= a->cols, "dropout: rows of %s overlap", name);
    return TDGS_OK;
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

int tdgs_dropout_apply(void* stream_, const tdgs_dropout* a) {
    TDGS_REQUIRE(a != nullptr, "dropout: null arguments");
    TDGS_REQUIRE(known_dtype(a->dtype), "dropout: unknown element type %d", a->dtype);
    TDGS_REQUIRE(a->rows >= 0 && a->cols >= 0 && (a->rows == 0 || a->cols <= INT64_MAX / 16 / a->rows),
                 "dropout: %lld rows of %lld", (long long)a->rows, (long long)a->cols);
    TDGS_REQUIRE(a->p >= 0.0 && a->p <= 1.0, "dropout: the probability is not in 0 to 1");
    if (a->rows == 0 || a->cols == 0) return TDGS_OK;
    TDGS_TRY(dr_check_rows(&a->x, "x", a, false));
    TDGS_TRY(dr_check_rows(&a->out, "out", a, true));
    if (a->residual.data) TDGS_TRY(dr_check_rows(&a->residual, "residual", a, false));
    auto bytes = [&](const tdgs_rows& v) {
        const int64_t size = (int64_t)dtype_size(a->dtype);
        return ByteRows(v.data, v.data ? a->rows : 0, a->rows > 1 ? v.stride * size : 0, a->cols * size);
    };
    TDGS_REQUIRE(same_or_apart(bytes(a->out), bytes(a->x)), "dropout: out overlaps x without being it");
    TDGS_REQUIRE(same_or_apart(bytes(a->out), bytes(a->residual)), "dropout: out overlaps the residual without being it");
    TDGS_REQUIRE(aligned_to(a->call_dev, 8), "dropout: the device's count of calls is not aligned");
    DrArgs r = {};
    r.x = a->x.data;
    r.residual = a->residual.data;
    r.out = a->out.data;
    r.xs = a->x.stride;
    r.rs = a->residual.stride;
    r.os = a->out.stride;
    r.rows = a->rows;
    r.cols = a->cols;
    r.key = PhiloxKey(a->seed);
    r.call = a->call;
    r.call_dev = a->call_dev;
    r.rule = DropRule(a->p);
    if (r.rows == 1 || (r.xs == r.cols && r.os == r.cols && (!r.residual || r.rs == r.cols))) {
        r.cols *= r.rows;
        r.rows = 1;
    }
    // whole words of the generator where every row starts on a multiple of four elements
    const int vw = r.rows > 1 && r.cols % 4 != 0 ? 1 : (a->dtype == TDGS_F32 || (r.rows > 1 && r.cols % 8 != 0) ? 4 : 8);
    const int64_t vectors = ceil_div(r.cols, vw);
    while (r.row_shift < 8 && ((int64_t)1 << r.row_shift) < vectors) ++r.row_shift;
    const int64_t across = ceil_div(vectors, (int64_t)1 << r.row_shift), down = ceil_div(r.rows, kDrThreads >> r.row_shift);
    const dim3 grid((unsigned)(across < (1 << 20) ? across : 1 << 20), (unsigned)(down < 65535 ? down : 65535));
    hipStream_t stream = (hipStream_t)stream_;
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (vw == 1) k_dropout<T, 1><<<grid, kDrThreads, 0, stream>>>(r);
        else if (vw == 4) k_dropout<T, 4><<<grid, kDrThreads, 0, stream>>>(r);
        else if constexpr (sizeof(T) == 2) k_dropout<T, 8><<<grid, kDrThreads, 0, stream>>>(r);
        TDGS_LAUNCHED();
        return TDGS_OK;
    });
}

}  // extern "C"
