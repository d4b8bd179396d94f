// norm.hip — group norm with an activation over channels-last images, forward and backward.
//
// A workgroup takes a run of pixels and all channels (or 256 vectors of them): thread t holds VW
// neighbouring channels, 16 bytes where the tensors allow it, of every (256 / vectors)th pixel, so
// its channels' statistics, weights and sums live in its registers and a pixel's channels are read
// as one contiguous piece. The kernels are bound by memory.
//
// Statistics are Welford's running mean and sum of squared deviations in 32 bits, per channel, and
// are joined between threads, workgroups and a group's channels by the exact rule for two parts
// (Chan, Golub & LeVeque 1979) in its form for many: mean = sum n_i mean_i / n,
// M2 = sum M2_i + n_i (mean_i - mean)^2. A sum of squares minus the squared mean would lose the variance of
// a channel whose mean is large.
//
// Three launches (runs of pixels, their joining, the result), or one for images of few pixels, a
// workgroup then taking all pixels of a few whole groups. 960x540x128 bfloat16 with SiLU: statistics 24 us (133 MB,
// 5.6 TB/s), joining 6 (latency), result 49 (265 MB, 5.4 TB/s): a large copy reaches 5.1, and the image just fits
// the last-level cache; 94 us together where every pass has another image. Reading it once only would take a wait of
// all workgroups for each other in the middle.
#include "internal.hpp"
#include "elem.hpp"
#include "activation.hpp"

namespace tdgs {

constexpr int kGnThreads = 256;
constexpr int kGnSmallThreads = 512;   // of a workgroup that takes whole groups, and
constexpr int kGnSmallVectors = 64;    // the most channel vectors it takes

struct GnArgs {
    const void *x, *dout, *weight, *bias;
    void *out, *dx, *dweight, *dbias;
    int64_t xn, xp, on, op, dn, dp, gn, gp;   // strides of x, out, dout, dx between images and pixels
    float* stats;                             // mean and 1 / deviation per image and group
    float *part, *chan;
    int64_t pixels, per;                      // per: pixels per workgroup
    int32_t n, channels, groups, group_size, blocks, vectors;
    int32_t parts;      // partial statistics per run: one per group, or per channel
    float eps;
    bool param_f32;
};

// Channel c's weight or bias (null: none given).
template <class T>
__device__ __forceinline__ float gn_param(const void* p, bool f32, int c, float none) {
    if (!p) return none;
    return f32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
}
template <class T>
__device__ __forceinline__ void gn_set_param(void* p, bool f32, int c, float v) {
    if (f32) ((float*)p)[c] = v;
    else ((T*)p)[c] = (T)v;
}

template <class T, int VW>
struct GnVec {
    typedef T V __attribute__((ext_vector_type(VW)));
    float f[VW];
    __device__ __forceinline__ void load(const T* __restrict__ p) {
        if constexpr (VW == 1) {
            f[0] = (float)*p;
        } else {
            const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
            for (int i = 0; i < VW; ++i) f[i] = (float)v[i];
        }
    }
    // Past the caches, which are to keep what an earlier pass has read for this one (960x540x128 bfloat16 101 -> 94 us).
    __device__ __forceinline__ void store(T* __restrict__ p) const {
        if constexpr (VW == 1) {
            *p = (T)f[0];
        } else {
            V v;
#pragma unroll
            for (int i = 0; i < VW; ++i) v[i] = (T)f[i];
            __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
        }
    }
};

// Where a thread of a workgroup of THREADS stands among `vectors` channel vectors.
template <int THREADS>
struct GnPlace {
    int cv, pl, lanes;   // channel vector, first pixel, pixels apart
    bool on;
    __device__ __forceinline__ explicit GnPlace(int vectors) {
        lanes = THREADS / vectors;
        cv = (int)threadIdx.x % vectors;
        pl = (int)threadIdx.x / vectors;
        on = pl < lanes;
    }
};

__device__ __forceinline__ float gn_segment_sum(float x, int width) {
    for (int w = width / 2; w > 0; w >>= 1) x += __shfl_xor(x, w, kWave);
    return x;
}

// Per-channel statistics of pixels [p0, p1) of the channels from x on, joined over the workgroup's
// lanes: thread c < vectors * VW leaves channel c's mean and sum of squared deviations in s_mean[c], s_m2[c].
template <class T, int VW, int THREADS>
__device__ __forceinline__ void gn_stats(const T* __restrict__ x, int64_t xp, int64_t p0, int64_t p1, int vectors,
                                         float* s_mean, float* s_m2) {
    const GnPlace<THREADS> at(vectors);
    float mean[VW], m2[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) mean[i] = m2[i] = 0.0f;
    if (at.on) {
        float count = 0.0f;
        constexpr int U = 4;
        int64_t p = p0 + at.pl;
        auto add = [&](const GnVec<T, VW>& v) {
            count += 1.0f;
            const float r = __builtin_amdgcn_rcpf(count);
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float d = v.f[i] - mean[i];
                mean[i] = __builtin_fmaf(d, r, mean[i]);
                m2[i] = __builtin_fmaf(d, v.f[i] - mean[i], m2[i]);
            }
        };
        for (; p + (U - 1) * at.lanes < p1; p += U * at.lanes) {
            GnVec<T, VW> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u].load(x + (p + u * at.lanes) * xp + at.cv * VW);
#pragma unroll
            for (int u = 0; u < U; ++u) add(v[u]);
        }
        for (; p < p1; p += at.lanes) {
            GnVec<T, VW> v;
            v.load(x + p * xp + at.cv * VW);
            add(v);
        }
    }
    // channel-major, the lanes of a channel next to each other and padded by one
    const int pitch = at.lanes | 1;
    if (at.on) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            s_mean[(at.cv * VW + i) * pitch + at.pl] = mean[i];
            s_m2[(at.cv * VW + i) * pitch + at.pl] = m2[i];
        }
    }
    __syncthreads();
    // `width` lanes per channel, a power of two up to a wavefront; each adds every width-th entry
    const int channels = vectors * VW;
    int width = 1;
    while (width < kWave && width * 2 <= at.lanes && width * 2 * channels <= THREADS) width *= 2;
    const int64_t pixels = p1 - p0;
    const int whole = (int)(pixels / at.lanes), extra = (int)(pixels % at.lanes);
    const int sub = (int)threadIdx.x & (width - 1);
    float out_m[VW], out_s[VW];
#pragma unroll
    for (int k = 0; k < VW; ++k) {
        const int c = (k * THREADS + (int)threadIdx.x) / width;
        out_m[k] = out_s[k] = 0.0f;
        if (k * THREADS / width >= channels) continue;
        float m = 0.0f, s2 = 0.0f;
        if (c < channels)
            for (int l = sub; l < at.lanes; l += width)
                m = __builtin_fmaf((float)(whole + (l < extra)), s_mean[c * pitch + l], m);
        m = gn_segment_sum(m, width) / (float)pixels;
        if (c < channels)
            for (int l = sub; l < at.lanes; l += width) {
                const float d = s_mean[c * pitch + l] - m;
                s2 += __builtin_fmaf((float)(whole + (l < extra)) * d, d, s_m2[c * pitch + l]);
            }
        out_m[k] = m;
        out_s[k] = gn_segment_sum(s2, width);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VW; ++k) {
        const int c = (k * THREADS + (int)threadIdx.x) / width;
        if (sub == 0 && c < channels) {
            s_mean[c] = out_m[k];
            s_m2[c] = out_s[k];
        }
    }
    __syncthreads();
}

// The statistics of `groups` groups of `size` channels, each channel over `pixels` pixels, from the
// channels' in LDS: f(group, mean, sum of squared deviations) by one lane each.
template <class F>
__device__ __forceinline__ void gn_groups(const float* s_mean, const float* s_m2, int groups, int size, float pixels,
                                          int threads, F&& f) {
    int width = 1;
    while (width < kWave && width < size) width *= 2;
    const int sub = (int)threadIdx.x & (width - 1);
    for (int g0 = 0; g0 < groups; g0 += threads / width) {
        const int g = g0 + (int)threadIdx.x / width;
        float m = 0.0f, s2 = 0.0f;
        if (g < groups)
            for (int c = sub; c < size; c += width) m += s_mean[g * size + c];
        m = gn_segment_sum(m, width) / (float)size;
        if (g < groups)
            for (int c = sub; c < size; c += width) {
                const float d = s_mean[g * size + c] - m;
                s2 += __builtin_fmaf(pixels * d, d, s_m2[g * size + c]);
            }
        s2 = gn_segment_sum(s2, width);
        if (g < groups && sub == 0) f(g, m, s2);
    }
}

__device__ __forceinline__ float gn_inverse(const GnArgs& a, float m2, float count) {
    return 1.0f / sqrtf(m2 / count + a.eps);
}

// Floats of LDS for one array of gn_stats or gn_sums: an entry per lane and channel, a channel's entries
// padded to an odd number (by a half at most, where there are two lanes).
template <int VW, int THREADS>
constexpr int gn_lds() { return VW * THREADS * 3 / 2; }

// Workgroup (b, y, n): statistics of run b of image n's pixels, channel block y; per group where a
// workgroup holds all channels (which a.parts does not tell: it is groups and channels in one for groups of one channel).
template <class T, int VW>
__global__ __launch_bounds__(kGnThreads) void k_norm_stats(GnArgs a) {
    __shared__ float s_mean[gn_lds<VW, kGnThreads>()];
    __shared__ float s_m2[gn_lds<VW, kGnThreads>()];
    const int b = blockIdx.x, n = blockIdx.z, v0 = blockIdx.y * kGnThreads;
    const int vectors = min(a.vectors - v0, kGnThreads), c0 = v0 * VW;
    const int64_t p0 = b * a.per, p1 = min(a.pixels, p0 + a.per);
    gn_stats<T, VW, kGnThreads>((const T*)a.x + n * a.xn + c0, a.xp, p0, p1, vectors, s_mean, s_m2);
    float2* const out = (float2*)a.part + ((int64_t)n * a.blocks + b) * a.parts;
    if (a.vectors <= kGnThreads) {
        gn_groups(s_mean, s_m2, a.groups, a.group_size, (float)(p1 - p0), kGnThreads,
                  [&](int g, float m, float s2) { out[g] = make_float2(m, s2); });
    } else {
        for (int c = threadIdx.x; c < vectors * VW; c += kGnThreads) out[c0 + c] = make_float2(s_mean[c], s_m2[c]);
    }
}

__device__ __forceinline__ float gn_block_sum(float x, float* s) {
    for (int w = kWave / 2; w > 0; w >>= 1) x += __shfl_xor(x, w, kWave);
    __syncthreads();
    if (__lane_id() == 0) s[threadIdx.x / kWave] = x;
    __syncthreads();
    float all = 0.0f;
    for (int w = 0; w < kGnThreads / kWave; ++w) all += s[w];
    return all;
}

// Workgroup n * groups + g: joins the runs (and the channels, where they came by channel) of a group.
static __global__ __launch_bounds__(kGnThreads) void k_norm_join(GnArgs a) {
    __shared__ float s[kGnThreads / kWave];
    const int n = blockIdx.x / a.groups, g = blockIdx.x % a.groups;
    const int size = a.parts == a.groups ? 1 : a.group_size;   // entries per run
    const float2* const part = (const float2*)a.part + (int64_t)n * a.blocks * a.parts + g * size;
    const float share = (float)(a.group_size / size);          // channels per entry
    const int64_t items = (int64_t)a.blocks * size;
    const float total = (float)a.pixels * (float)a.group_size;
    auto each = [&](auto&& f) {
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < items; i += kGnThreads) {
            const int b = size == 1 ? (int)i : (int)(i / size), c = size == 1 ? 0 : (int)(i % size);
            f(part[(int64_t)b * a.parts + c], share * (float)(min(a.pixels, (b + 1) * a.per) - b * a.per));
        }
    };
    float m = 0.0f, m2 = 0.0f;
    each([&](const float2& v, float count) { m = __builtin_fmaf(count, v.x, m); });
    m = gn_block_sum(m, s) / total;
    each([&](const float2& v, float count) {
        const float d = v.x - m;
        m2 += __builtin_fmaf(count * d, d, v.y);
    });
    m2 = gn_block_sum(m2, s);
    if (threadIdx.x == 0) {
        a.stats[2 * blockIdx.x] = m;
        a.stats[2 * blockIdx.x + 1] = gn_inverse(a, m2, total);
    }
}

// What a thread needs of its channels: xhat = (x - mean) r, z = xhat w + b.
template <class T, int VW>
struct GnChannels {
    float mean[VW], r[VW], w[VW], b[VW];
    // stats: of the groups from g0 on
    __device__ __forceinline__ void load(const GnArgs& a, const float* stats, int c0, int g0 = 0) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const int g = (c0 + i) / a.group_size - g0;
            mean[i] = stats[2 * g];
            r[i] = stats[2 * g + 1];
            w[i] = gn_param<T>(a.weight, a.param_f32, c0 + i, 1.0f);
            b[i] = gn_param<T>(a.bias, a.param_f32, c0 + i, 0.0f);
        }
    }
};

template <class T, int VW, int ACT, int THREADS>
__device__ __forceinline__ void gn_apply(const GnArgs& a, const T* __restrict__ x, T* __restrict__ out,
                                         const GnChannels<T, VW>& ch, int64_t p0, int64_t p1,
                                         const GnPlace<THREADS>& at) {
    float rw[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) rw[i] = ch.r[i] * ch.w[i];
    auto one = [&](GnVec<T, VW>& v) {
        float none;
#pragma unroll
        for (int i = 0; i < VW; ++i)
            v.f[i] = act_value<ACT, false>(__builtin_fmaf(v.f[i] - ch.mean[i], rw[i], ch.b[i]), &none);
    };
    constexpr int U = 4;
    int64_t p = p0 + at.pl;
    for (; p + (U - 1) * at.lanes < p1; p += U * at.lanes) {
        GnVec<T, VW> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load(x + (p + u * at.lanes) * a.xp + at.cv * VW);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            one(v[u]);
            v[u].store(out + (p + u * at.lanes) * a.op + at.cv * VW);
        }
    }
    for (; p < p1; p += at.lanes) {
        GnVec<T, VW> v;
        v.load(x + p * a.xp + at.cv * VW);
        one(v);
        v.store(out + p * a.op + at.cv * VW);
    }
}

template <class T, int VW, int ACT>
__global__ __launch_bounds__(kGnThreads) void k_norm_apply(GnArgs a) {
    const int b = blockIdx.x, n = blockIdx.z, v0 = blockIdx.y * kGnThreads, c0 = v0 * VW;
    const GnPlace<kGnThreads> at(min(a.vectors - v0, kGnThreads));
    if (!at.on) return;
    GnChannels<T, VW> ch;
    ch.load(a, a.stats + (int64_t)2 * n * a.groups, c0 + at.cv * VW);
    const int64_t p0 = b * a.per, p1 = min(a.pixels, p0 + a.per);
    gn_apply<T, VW, ACT, kGnThreads>(a, (const T*)a.x + n * a.xn + c0, (T*)a.out + n * a.on + c0, ch, p0, p1, at);
}

// Workgroup (y, n): all pixels of channel block y, whole groups of a.vectors vectors, of image n. 8x8x128 floats: 5.8 us,
// the latency of one load, the joining and one store (three launches: 10.7).
template <class T, int VW, int ACT>
__global__ __launch_bounds__(kGnSmallThreads) void k_norm_small(GnArgs a) {
    __shared__ float s_mean[gn_lds<VW, kGnSmallThreads>()];
    __shared__ float s_m2[gn_lds<VW, kGnSmallThreads>()];
    __shared__ float s_stats[2 * kGnSmallVectors * VW];
    const int n = blockIdx.y, c0 = blockIdx.x * a.vectors * VW, g0 = c0 / a.group_size;
    const int vectors = min(a.vectors, a.channels / VW - (int)blockIdx.x * a.vectors);
    const T* const x = (const T*)a.x + n * a.xn + c0;
    gn_stats<T, VW, kGnSmallThreads>(x, a.xp, 0, a.pixels, vectors, s_mean, s_m2);
    float* const stats = a.stats ? a.stats + ((int64_t)n * a.groups + g0) * 2 : nullptr;
    gn_groups(s_mean, s_m2, vectors * VW / a.group_size, a.group_size, (float)a.pixels, kGnSmallThreads,
              [&](int g, float m, float s2) {
                  const float r = gn_inverse(a, s2, (float)a.pixels * (float)a.group_size);
                  s_stats[2 * g] = m;
                  s_stats[2 * g + 1] = r;
                  if (stats) {
                      stats[2 * g] = m;
                      stats[2 * g + 1] = r;
                  }
              });
    __syncthreads();
    const GnPlace<kGnSmallThreads> at(vectors);
    if (!at.on) return;
    GnChannels<T, VW> ch;
    ch.load(a, s_stats, c0 + at.cv * VW, g0);
    gn_apply<T, VW, ACT, kGnSmallThreads>(a, x, (T*)a.out + n * a.on + c0, ch, 0, a.pixels, at);
}

// ---- backward ------------------------------------------------------------------------------

// e = dout act'(z) and xhat of one vector.
template <class T, int VW, int ACT>
__device__ __forceinline__ void gn_slope(const GnChannels<T, VW>& ch, const GnVec<T, VW>& x, const GnVec<T, VW>& d,
                                         float (&e)[VW], float (&xhat)[VW]) {
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        float slope;
        xhat[i] = (x.f[i] - ch.mean[i]) * ch.r[i];
        act_value<ACT, true>(__builtin_fmaf(xhat[i], ch.w[i], ch.b[i]), &slope);
        e[i] = d.f[i] * slope;
    }
}

// Sums of e and e xhat over pixels [p0, p1), per channel, joined over the workgroup's lanes into
// s_1[channel] and s_2[channel].
template <class T, int VW, int ACT, int THREADS>
__device__ __forceinline__ void gn_sums(const GnArgs& a, const T* __restrict__ x, const T* __restrict__ dout,
                                        const GnChannels<T, VW>& ch, int64_t p0, int64_t p1,
                                        const GnPlace<THREADS>& at, int vectors, float* s_1, float* s_2) {
    const int pitch = at.lanes | 1;
    if (at.on) {
        float s1[VW], s2[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) s1[i] = s2[i] = 0.0f;
        auto add = [&](const GnVec<T, VW>& vx, const GnVec<T, VW>& vd) {
            float e[VW], xhat[VW];
            gn_slope<T, VW, ACT>(ch, vx, vd, e, xhat);
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                s1[i] += e[i];
                s2[i] = __builtin_fmaf(e[i], xhat[i], s2[i]);
            }
        };
        constexpr int U = 2;
        int64_t p = p0 + at.pl;
        for (; p + (U - 1) * at.lanes < p1; p += U * at.lanes) {
            GnVec<T, VW> vx[U], vd[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                vx[u].load(x + (p + u * at.lanes) * a.xp + at.cv * VW);
                vd[u].load(dout + (p + u * at.lanes) * a.dp + at.cv * VW);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) add(vx[u], vd[u]);
        }
        for (; p < p1; p += at.lanes) {
            GnVec<T, VW> vx, vd;
            vx.load(x + p * a.xp + at.cv * VW);
            vd.load(dout + p * a.dp + at.cv * VW);
            add(vx, vd);
        }
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            s_1[(at.cv * VW + i) * pitch + at.pl] = s1[i];
            s_2[(at.cv * VW + i) * pitch + at.pl] = s2[i];
        }
    }
    __syncthreads();
    const int channels = vectors * VW;
    int width = 1;
    while (width < kWave && width * 2 <= at.lanes && width * 2 * channels <= THREADS) width *= 2;
    const int sub = (int)threadIdx.x & (width - 1);
    float o1[VW], o2[VW];
#pragma unroll
    for (int k = 0; k < VW; ++k) {
        const int c = (k * THREADS + (int)threadIdx.x) / width;
        o1[k] = o2[k] = 0.0f;
        if (k * THREADS / width >= channels) continue;
        if (c < channels)
            for (int l = sub; l < at.lanes; l += width) {
                o1[k] += s_1[c * pitch + l];
                o2[k] += s_2[c * pitch + l];
            }
        o1[k] = gn_segment_sum(o1[k], width);
        o2[k] = gn_segment_sum(o2[k], width);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VW; ++k) {
        const int c = (k * THREADS + (int)threadIdx.x) / width;
        if (sub == 0 && c < channels) {
            s_1[c] = o1[k];
            s_2[c] = o2[k];
        }
    }
    __syncthreads();
}

template <class T, int VW, int ACT>
__global__ __launch_bounds__(kGnThreads) void k_norm_sums(GnArgs a) {
    __shared__ float s_1[gn_lds<VW, kGnThreads>()];
    __shared__ float s_2[gn_lds<VW, kGnThreads>()];
    const int b = blockIdx.x, n = blockIdx.z, v0 = blockIdx.y * kGnThreads, c0 = v0 * VW;
    const int vectors = min(a.vectors - v0, kGnThreads);
    const GnPlace<kGnThreads> at(vectors);
    GnChannels<T, VW> ch;
    ch.load(a, a.stats + (int64_t)2 * n * a.groups, c0 + at.cv * VW);
    const int64_t p0 = b * a.per, p1 = min(a.pixels, p0 + a.per);
    gn_sums<T, VW, ACT, kGnThreads>(a, (const T*)a.x + n * a.xn + c0, (const T*)a.dout + n * a.dn + c0, ch, p0, p1, at,
                                    vectors, s_1, s_2);
    float2* const out = (float2*)a.part + ((int64_t)n * a.blocks + b) * a.channels + c0;
    for (int c = threadIdx.x; c < vectors * VW; c += kGnThreads) out[c] = make_float2(s_1[c], s_2[c]);
}

// Workgroup (y, n): 8 channels of image n, joins the runs to chan.
static __global__ __launch_bounds__(kGnThreads) void k_norm_sums_join(GnArgs a) {
    constexpr int C = 8, L = kGnThreads / C;
    __shared__ float2 s[L][C + 1];
    const int cc = threadIdx.x % C, c = blockIdx.x * C + cc, lane = threadIdx.x / C, n = blockIdx.y;
    float2 v = make_float2(0.0f, 0.0f);
    if (c < a.channels) {
        const float2* const part = (const float2*)a.part + (int64_t)n * a.blocks * a.channels + c;
#pragma unroll 4
        for (int b = lane; b < a.blocks; b += L) {
            const float2 p = part[(int64_t)b * a.channels];
            v.x += p.x;
            v.y += p.y;
        }
    }
    s[lane][cc] = v;
    for (int w = L / 2; w > 0; w >>= 1) {
        __syncthreads();
        if (lane < w) {
            s[lane][cc].x += s[lane + w][cc].x;
            s[lane][cc].y += s[lane + w][cc].y;
        }
    }
    if (lane == 0 && c < a.channels) ((float2*)a.chan)[(int64_t)n * a.channels + c] = s[0][cc];
}

// Thread per channel: the images' sums to dbias and dweight.
template <class T>
__device__ __forceinline__ void gn_params(const GnArgs& a, int c) {
    float db = 0.0f, dw = 0.0f;
    for (int n = 0; n < a.n; ++n) {
        const float2 v = ((const float2*)a.chan)[(int64_t)n * a.channels + c];
        db += v.x;
        dw += v.y;
    }
    if (a.dweight) gn_set_param<T>(a.dweight, a.param_f32, c, dw);
    if (a.dbias) gn_set_param<T>(a.dbias, a.param_f32, c, db);
}

template <class T>
__global__ __launch_bounds__(kGnThreads) void k_norm_params(GnArgs a) {
    const int c = blockIdx.x * kGnThreads + threadIdx.x;
    if (c < a.channels) gn_params<T>(a, c);
}

// dx of pixels [p0, p1): r (w e - m1 - xhat m2), m1 and m2 the group's means of w e and w e xhat.
template <class T, int VW, int ACT, int THREADS>
__device__ __forceinline__ void gn_dx(const GnArgs& a, const T* __restrict__ x, const T* __restrict__ dout,
                                      T* __restrict__ dx, const GnChannels<T, VW>& ch, const float (&m1)[VW],
                                      const float (&m2)[VW], int64_t p0, int64_t p1, const GnPlace<THREADS>& at) {
    auto one = [&](const GnVec<T, VW>& vx, GnVec<T, VW>& vd) {
        float e[VW], xhat[VW];
        gn_slope<T, VW, ACT>(ch, vx, vd, e, xhat);
#pragma unroll
        for (int i = 0; i < VW; ++i)
            vd.f[i] = ch.r[i] * __builtin_fmaf(-xhat[i], m2[i], __builtin_fmaf(ch.w[i], e[i], -m1[i]));
    };
    constexpr int U = 2;
    int64_t p = p0 + at.pl;
    for (; p + (U - 1) * at.lanes < p1; p += U * at.lanes) {
        GnVec<T, VW> vx[U], vd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vx[u].load(x + (p + u * at.lanes) * a.xp + at.cv * VW);
            vd[u].load(dout + (p + u * at.lanes) * a.dp + at.cv * VW);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            one(vx[u], vd[u]);
            vd[u].store(dx + (p + u * at.lanes) * a.gp + at.cv * VW);
        }
    }
    for (; p < p1; p += at.lanes) {
        GnVec<T, VW> vx, vd;
        vx.load(x + p * a.xp + at.cv * VW);
        vd.load(dout + p * a.dp + at.cv * VW);
        one(vx, vd);
        vd.store(dx + p * a.gp + at.cv * VW);
    }
}

// A group's means of w e and w e xhat, from its channels' sums, by one wavefront.
template <class T, class Sum>
__device__ __forceinline__ float2 gn_group_means(const GnArgs& a, int g, Sum&& sum) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = g * a.group_size + (int)__lane_id(); c < (g + 1) * a.group_size; c += kWave) {
        const float w = gn_param<T>(a.weight, a.param_f32, c, 1.0f);
        const float2 v = sum(c);
        s1 = __builtin_fmaf(w, v.x, s1);
        s2 = __builtin_fmaf(w, v.y, s2);
    }
    const float count = (float)a.pixels * (float)a.group_size;
    return make_float2(gn_segment_sum(s1, kWave) / count, gn_segment_sum(s2, kWave) / count);
}

// The first workgroups also write dbias and dweight. 3 x 33565 x 96 floats: 21 us (116 MB, 5.4 TB/s), the sums before it
// 16 (77 MB, 4.9 TB/s).
template <class T, int VW, int ACT>
__global__ __launch_bounds__(kGnThreads) void k_norm_dx(GnArgs a) {
    __shared__ float2 s_means[kGnThreads * VW];
    const int b = blockIdx.x, n = blockIdx.z, v0 = blockIdx.y * kGnThreads, c0 = v0 * VW;
    const int vectors = min(a.vectors - v0, kGnThreads);
    if (b == 0 && n == 0)
        for (int c = threadIdx.x; c < vectors * VW; c += kGnThreads) gn_params<T>(a, c0 + c);
    const int g0 = c0 / a.group_size, g1 = (c0 + vectors * VW - 1) / a.group_size;
    for (int g = g0 + threadIdx.x / kWave; g <= g1; g += kGnThreads / kWave) {
        const float2 m = gn_group_means<T>(
            a, g, [&](int c) { return ((const float2*)a.chan)[(int64_t)n * a.channels + c]; });
        if (__lane_id() == 0) s_means[g - g0] = m;
    }
    __syncthreads();
    const GnPlace<kGnThreads> at(vectors);
    if (!at.on) return;
    GnChannels<T, VW> ch;
    ch.load(a, a.stats + (int64_t)2 * n * a.groups, c0 + at.cv * VW);
    float m1[VW], m2[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        const float2 m = s_means[(c0 + at.cv * VW + i) / a.group_size - g0];
        m1[i] = m.x;
        m2[i] = m.y;
    }
    const int64_t p0 = b * a.per, p1 = min(a.pixels, p0 + a.per);
    gn_dx<T, VW, ACT, kGnThreads>(a, (const T*)a.x + n * a.xn + c0, (const T*)a.dout + n * a.dn + c0,
                                  (T*)a.dx + n * a.gn + c0, ch, m1, m2, p0, p1, at);
}

// Workgroup (y, n): all pixels of channel block y of image n. dbias and dweight too for a single image;
// otherwise the sums go to chan.
template <class T, int VW, int ACT>
__global__ __launch_bounds__(kGnSmallThreads) void k_norm_small_grad(GnArgs a) {
    __shared__ float s_1[gn_lds<VW, kGnSmallThreads>()];
    __shared__ float s_2[gn_lds<VW, kGnSmallThreads>()];
    __shared__ float2 s_means[kGnSmallVectors * VW];
    const int n = blockIdx.y, c0 = blockIdx.x * a.vectors * VW, g0 = c0 / a.group_size;
    const int vectors = min(a.vectors, a.channels / VW - (int)blockIdx.x * a.vectors);
    const GnPlace<kGnSmallThreads> at(vectors);
    const T* const x = (const T*)a.x + n * a.xn + c0;
    const T* const dout = (const T*)a.dout + n * a.dn + c0;
    GnChannels<T, VW> ch;
    ch.load(a, a.stats + (int64_t)2 * n * a.groups, c0 + at.cv * VW);
    gn_sums<T, VW, ACT, kGnSmallThreads>(a, x, dout, ch, 0, a.pixels, at, vectors, s_1, s_2);
    for (int c = threadIdx.x; c < vectors * VW; c += kGnSmallThreads) {
        if (a.n > 1) {
            ((float2*)a.chan)[(int64_t)n * a.channels + c0 + c] = make_float2(s_1[c], s_2[c]);
        } else {
            if (a.dweight) gn_set_param<T>(a.dweight, a.param_f32, c0 + c, s_2[c]);
            if (a.dbias) gn_set_param<T>(a.dbias, a.param_f32, c0 + c, s_1[c]);
        }
    }
    for (int g = g0 + threadIdx.x / kWave; g * a.group_size < c0 + vectors * VW; g += kGnSmallThreads / kWave) {
        const float2 m = gn_group_means<T>(a, g, [&](int c) { return make_float2(s_1[c - c0], s_2[c - c0]); });
        if (__lane_id() == 0) s_means[g - g0] = m;
    }
    __syncthreads();
    if (!at.on) return;
    float m1[VW], m2[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        const float2 m = s_means[(c0 + at.cv * VW + i) / a.group_size - g0];
        m1[i] = m.x;
        m2[i] = m.y;
    }
    gn_dx<T, VW, ACT, kGnSmallThreads>(a, x, dout, (T*)a.dx + n * a.gn + c0, ch, m1, m2, 0, a.pixels, at);
}

// ---- host ----------------------------------------------------------------------------------

struct GnPlan {
    int vw, vectors, blocks, parts;
    int64_t per;
    bool small;            // one launch, a workgroup per `vectors` vectors of whole groups
    size_t stats_bytes, chan_bytes;
    size_t forward_bytes, grad_bytes;
};

// Workgroups of one pass over all images, and the least pixels a thread takes: the runs' joining costs
// as much as they are many.
constexpr int64_t kGnWorkgroups = 1024;
constexpr int64_t kGnPixels = 8;
// Pixels per thread up to which one launch is taken.
constexpr int64_t kGnSmallPixels = 16;

static GnPlan gn_plan(const tdgs_norm* a, bool vec) {
    GnPlan p;
    p.vw = vec ? (a->dtype == TDGS_F32 ? 4 : 8) : 1;
    p.vectors = a->channels / p.vw;
    p.stats_bytes = align_up((size_t)a->n * a->groups * 2 * sizeof(float));
    p.chan_bytes = align_up((size_t)a->n * a->channels * 2 * sizeof(float));
    // whole groups in whole vectors, 64 bytes of a pixel or more
    const int size = a->channels / a->groups;
    int unit = size;
    while (unit % p.vw != 0) unit += size;
    unit /= p.vw;
    const int least = vec ? 4 : (int)(64 / dtype_size(a->dtype));
    int few = (least + unit - 1) / unit * unit;
    if (few > p.vectors) few = p.vectors;
    p.small = few <= kGnSmallVectors && a->pixels <= kGnSmallPixels * (kGnSmallThreads / few);
    if (p.small) {
        p.vectors = few;
        p.blocks = 1;
        p.parts = 0;
        p.per = a->pixels;
        p.forward_bytes = 0;
        p.grad_bytes = p.chan_bytes;
        return p;
    }
    const int64_t lanes = p.vectors < kGnThreads ? kGnThreads / p.vectors : 1;
    int64_t blocks = ceil_div(a->pixels, lanes * kGnPixels);
    const int64_t most = ceil_div(kGnWorkgroups, (a->n > 0 ? a->n : 1) * ceil_div(p.vectors, kGnThreads));
    if (blocks > most) blocks = most;
    p.per = ceil_div(a->pixels, blocks > 0 ? blocks : 1);
    p.blocks = (int)ceil_div(a->pixels, p.per > 0 ? p.per : 1);
    p.parts = p.vectors <= kGnThreads ? a->groups : a->channels;
    p.forward_bytes = p.stats_bytes + align_up((size_t)a->n * p.blocks * p.parts * 2 * sizeof(float));
    p.grad_bytes = p.chan_bytes + align_up((size_t)a->n * p.blocks * a->channels * 2 * sizeof(float));
    return p;
}

static int gn_check(const tdgs_norm* a) {
    TDGS_REQUIRE(a != nullptr, "group norm: null arguments");
    TDGS_REQUIRE(known_dtype(a->dtype), "group norm: unknown element type %d", a->dtype);
    TDGS_REQUIRE(a->param_dtype == a->dtype || a->param_dtype == TDGS_F32,
                 "group norm: weight and bias must be float32 or of the input's type");
    TDGS_REQUIRE(a->n >= 0 && a->pixels >= 0 && a->n <= 65535, "group norm: %d images of %lld pixels", a->n,
                 (long long)a->pixels);
    TDGS_REQUIRE(a->channels > 0 && a->channels <= (1 << 20) && a->groups > 0 && a->channels % a->groups == 0,
                 "group norm: %d channels do not divide into %d groups", a->channels, a->groups);
    TDGS_REQUIRE((int64_t)a->n * a->groups <= INT32_MAX, "group norm: %d groups in each of %d images", a->groups, a->n);
    TDGS_REQUIRE(a->activation >= TDGS_ACT_IDENTITY && a->activation <= TDGS_ACT_RELU, "group norm: unknown activation %d",
                 a->activation);
    TDGS_REQUIRE(a->eps >= 0.0f && a->eps < INFINITY, "group norm: eps must be finite and not negative");
    return TDGS_OK;
}

static int gn_check_view(const tdgs_pixels* v, const char* name, const tdgs_norm* a, bool written) {
    TDGS_REQUIRE(v->data != nullptr, "group norm: %s is null", name);
    TDGS_REQUIRE(aligned_to(v->data, (size_t)dtype_size(a->dtype)), "group norm: %s is not aligned to its element type", name);
    TDGS_REQUIRE(v->stride_n >= 0 && v->stride_p >= 0, "group norm: %s has a negative stride", name);
    if (written)
        TDGS_REQUIRE((a->n <= 1 || v->stride_n >= a->channels) && (a->pixels <= 1 || v->stride_p >= a->channels),
                     "group norm: pixels of %s overlap", name);
    return TDGS_OK;
}

static bool gn_vec(const tdgs_pixels& v, const tdgs_norm* a) {
    const int64_t e = dtype_size(a->dtype);
    return a->channels * e % 16 == 0 && aligned_to(v.data, 16) && v.stride_n * e % 16 == 0 && v.stride_p * e % 16 == 0;
}

static GnArgs gn_args(const tdgs_norm* a, const GnPlan& p) {
    GnArgs r = {};
    r.x = a->x.data;
    r.xn = a->x.stride_n;
    r.xp = a->x.stride_p;
    r.weight = a->weight;
    r.bias = a->bias;
    r.stats = a->stats;
    r.pixels = a->pixels;
    r.per = p.per;
    r.n = a->n;
    r.channels = a->channels;
    r.groups = a->groups;
    r.group_size = a->channels / a->groups;
    r.blocks = p.blocks;
    r.vectors = p.vectors;
    r.parts = p.parts;
    r.eps = a->eps;
    r.param_f32 = a->param_dtype == TDGS_F32;
    return r;
}

// f(T{}, vector width, activation) for the call's kernels.
template <class F>
static int gn_dispatch(const tdgs_norm* a, int vw, F&& f) {
    return with_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        auto with_act = [&](auto w) -> int {
            switch (a->activation) {
                case TDGS_ACT_IDENTITY: return f(t, w, std::integral_constant<int, TDGS_ACT_IDENTITY>{});
                case TDGS_ACT_SILU: return f(t, w, std::integral_constant<int, TDGS_ACT_SILU>{});
                case TDGS_ACT_GELU: return f(t, w, std::integral_constant<int, TDGS_ACT_GELU>{});
                default: return f(t, w, std::integral_constant<int, TDGS_ACT_RELU>{});
            }
        };
        return vw == 1 ? with_act(std::integral_constant<int, 1>{}) : with_act(std::integral_constant<int, 16 / (int)sizeof(T)>{});
    });
}

}  // namespace tdgs

using namespace tdgs;

extern "C" {

size_t tdgs_group_norm_temp_bytes(const tdgs_norm* a, int32_t grad) {
    if (gn_check(a) != TDGS_OK) return 0;
    size_t bytes = 0;
    for (int vec = 0; vec < 2; ++vec) {
        if (vec && a->channels * dtype_size(a->dtype) % 16 != 0) continue;
        const GnPlan p = gn_plan(a, vec != 0);
        const size_t b = grad && p.grad_bytes > p.forward_bytes ? p.grad_bytes : p.forward_bytes;
        if (b > bytes) bytes = b;
    }
    return bytes;
}

int tdgs_group_norm(void* stream_, const tdgs_norm* a) {
    TDGS_TRY(gn_check(a));
    if (a->n == 0 || a->pixels == 0) return TDGS_OK;
    TDGS_TRY(gn_check_view(&a->x, "x", a, false));
    TDGS_TRY(gn_check_view(&a->out, "out", a, true));
    const bool vec = gn_vec(a->x, a) && gn_vec(a->out, a);
    const GnPlan p = gn_plan(a, vec);
    TDGS_REQUIRE(p.forward_bytes == 0 || (a->temp && a->temp_bytes >= p.forward_bytes && aligned_to(a->temp, 16)),
                 "group norm: scratch of %zu bytes, %zu needed", a->temp ? a->temp_bytes : (size_t)0, p.forward_bytes);
    hipStream_t stream = (hipStream_t)stream_;
    GnArgs r = gn_args(a, p);
    r.out = a->out.data;
    r.on = a->out.stride_n;
    r.op = a->out.stride_p;
    const dim3 small_grid((unsigned)ceil_div(a->channels / p.vw, p.vectors), (unsigned)a->n);
    if (!p.small) {
        if (!r.stats) r.stats = (float*)a->temp;
        r.part = (float*)((char*)a->temp + p.stats_bytes);
    }
    const dim3 grid((unsigned)p.blocks, (unsigned)ceil_div(p.vectors, kGnThreads), (unsigned)a->n);
    return gn_dispatch(a, p.vw, [&](auto t, auto w, auto act) -> int {
        using T = decltype(t);
        constexpr int VW = decltype(w)::value, ACT = decltype(act)::value;
        if (p.small) {
            k_norm_small<T, VW, ACT><<<small_grid, kGnSmallThreads, 0, stream>>>(r);
            TDGS_LAUNCHED();
            return TDGS_OK;
        }
        k_norm_stats<T, VW><<<grid, kGnThreads, 0, stream>>>(r);
        TDGS_LAUNCHED();
        k_norm_join<<<(unsigned)((int64_t)a->n * a->groups), kGnThreads, 0, stream>>>(r);
        TDGS_LAUNCHED();
        k_norm_apply<T, VW, ACT><<<grid, kGnThreads, 0, stream>>>(r);
        TDGS_LAUNCHED();
        return TDGS_OK;
    });
}

int tdgs_group_norm_grad(void* stream_, const tdgs_norm* a, const tdgs_norm_grads* g) {
    TDGS_TRY(gn_check(a));
    TDGS_REQUIRE(g != nullptr, "group norm: null gradients");
    TDGS_REQUIRE(a->stats != nullptr, "group norm: the gradient needs the forward call's stats");
    const bool empty = a->n == 0 || a->pixels == 0;
    if (!empty) {
        TDGS_TRY(gn_check_view(&a->x, "x", a, false));
        TDGS_TRY(gn_check_view(&g->dout, "dout", a, false));
        TDGS_TRY(gn_check_view(&g->dx, "dx", a, true));
    }
    const bool vec = !empty && gn_vec(a->x, a) && gn_vec(g->dout, a) && gn_vec(g->dx, a);
    const GnPlan p = gn_plan(a, vec);
    TDGS_REQUIRE(a->temp && a->temp_bytes >= p.grad_bytes && aligned_to(a->temp, 16),
                 "group norm: scratch of %zu bytes, the gradient needs %zu", a->temp ? a->temp_bytes : (size_t)0,
                 p.grad_bytes);
    hipStream_t stream = (hipStream_t)stream_;
    GnArgs r = gn_args(a, p);
    r.dout = g->dout.data;
    r.dn = g->dout.stride_n;
    r.dp = g->dout.stride_p;
    r.dx = g->dx.data;
    r.gn = g->dx.stride_n;
    r.gp = g->dx.stride_p;
    r.dweight = g->dweight;
    r.dbias = g->dbias;
    r.chan = (float*)a->temp;
    r.part = (float*)((char*)a->temp + p.chan_bytes);
    const dim3 small_grid((unsigned)ceil_div(a->channels / p.vw, p.vectors), (unsigned)a->n);
    const dim3 grid((unsigned)p.blocks, (unsigned)ceil_div(p.vectors, kGnThreads), (unsigned)a->n);
    return gn_dispatch(a, p.vw, [&](auto t, auto w, auto act) -> int {
        using T = decltype(t);
        constexpr int VW = decltype(w)::value, ACT = decltype(act)::value;
        const unsigned channel_blocks = (unsigned)ceil_div(a->channels, kGnThreads);
        if (empty) {
            r.n = 0;   // (dweight and dbias are zero)
            k_norm_params<T><<<channel_blocks, kGnThreads, 0, stream>>>(r);
            TDGS_LAUNCHED();
        } else if (p.small) {
            k_norm_small_grad<T, VW, ACT><<<small_grid, kGnSmallThreads, 0, stream>>>(r);
            TDGS_LAUNCHED();
            if (a->n > 1) {
                k_norm_params<T><<<channel_blocks, kGnThreads, 0, stream>>>(r);
                TDGS_LAUNCHED();
            }
        } else {
            k_norm_sums<T, VW, ACT><<<grid, kGnThreads, 0, stream>>>(r);
            TDGS_LAUNCHED();
            k_norm_sums_join<<<dim3((unsigned)ceil_div(a->channels, 8), (unsigned)a->n), kGnThreads, 0, stream>>>(r);
            TDGS_LAUNCHED();
            k_norm_dx<T, VW, ACT><<<grid, kGnThreads, 0, stream>>>(r);
            TDGS_LAUNCHED();
        }
        return TDGS_OK;
    });
}

}  // extern "C"
