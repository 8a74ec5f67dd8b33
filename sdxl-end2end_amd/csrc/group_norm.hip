// Group norm and its gradients (include/sdxl_hip/group_norm.h), for gfx950
// (MI355X, CDNA4).
//
// Bound by the tensor's bytes. Two launches a direction: the first one reads x
// (and dy) and leaves sums by chunk of pixels, the second one reads them again,
// out of the Infinity Cache where they fit it, and writes y (dx). A thread keeps
// to 16 bytes of channels (8 of a 16-bit type, 4 fp32 values) and goes down the
// pixels, so that a channel's constants and sums stay in registers and groups of
// any width (10, 20, 30 channels) cost nothing. A row's last 16 bytes may overlap
// the ones before them (any channel count from a vector up); what is there twice
// counts once.
//
// A workgroup owns a slab of whole groups, 512 bytes of every row or a little
// more, and a chunk of pixels: with full rows instead it would take as many
// chunks as workgroups, whose parts every workgroup of the second pass has to
// merge ([2, 4096, 960] fp16: 66 us, of which 256 chunks' parts were most).
//
// Statistics: a thread takes its pixels in batches of eight and sums x - p and (x - p)^2 of a batch, with p the mean of
// the pixels before it (of the first batch: its first value), then adds the batch to its mean and its sum M of squares
// about it. Summed about the first value alone, q of n pixels is up to n M where that value lies far from the others, and
// n roundings of such a q left M off by a relative n^2 2^-24 ([129, 16384, 128] fp32, 1024 pixels a thread, a first value
// 1000 deviations away: rstd off by 1.7e-3, so by 1.1e-6). About the mean so far a batch's q is at most twice what it adds to M (the first
// one's eight times). Parts {mean, M} of threads, then of chunks, are merged in the same way: by a lane about its own
// first part, M = sum M_i + n_i d_i^2 - (sum n_i d_i)^2 / n with d_i = mean_i - mean_0, of as many parts as it has (I of
// them: M off by a relative 3 (I + 1) (I + 3) 2^-24 at most), then over the lanes of its team about the mean of all.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "group_norm_device.hpp"
#include "int8_device.hpp"
#include "wave_reduce.hpp"

namespace sdxl_hip {
namespace {

constexpr int kMaxThreads = 512;

// The workgroup's slab: its first group, groups, first channel and channels.
struct GnSlab {
    int g0, groups, c0, channels;
};
__device__ __forceinline__ GnSlab slab_of(const GnParams& p, int slab) {
    const int g0 = slab * p.slab_groups;
    return {g0, p.slab_groups, g0 * p.group_channels, p.slab_groups * p.group_channels};
}

// The thread's place: row r of the rows at a time, first channel c0 of its vector in the slab, of which the first `skip`
// are the vector's before.
struct GnPlace {
    int r, c0, skip;
};
template <int kV>
__device__ __forceinline__ GnPlace place_of(const GnParams& p, const GnSlab& slab) {
    const int r = (int)threadIdx.x / p.vecs, v = (int)threadIdx.x % p.vecs;
    const int c0 = min(v * kV, slab.channels - kV);
    return {r, c0, v * kV - c0};
}

// The group of channel c (below 2^22: the quotient is at least half a step from the next integer).
__device__ __forceinline__ int group_of(const GnParams& p, int c) { return (int)(((float)c + 0.5f) * (1.0f / (float)p.group_channels)); }

// over a team of 16 lanes or of 64
__device__ __forceinline__ float team_sum(float v, int team) {
    v = reduce16(v, Add{});
    return team == 64 ? reduce_rows(v, Add{}) : v;
}

// pixels that row r of `rows` has of `count`
__device__ __forceinline__ int share_of(int count, int r, int rows) { return (count - r + rows - 1) / rows; }

// kBatch pixels' vectors of one tensor or two (b), on their way together. Past the `left` pixels that there are the last one
// is read again (none: the address itself, which has to be there): loads under conditions wait for each other, as they do
// without the scheduling barriers, between which the compiler takes them one by one to save registers ([1, 262144, 256]
// fp32, the first pass: 72 us so).
template <int kBatch, bool kTwo>
struct GnBatch {
    u32x4 a[kBatch], b[kTwo ? kBatch : 1];

    __device__ __forceinline__ void load(int left, const char* from_a, int64_t step_a, const char* from_b, int64_t step_b) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            a[k] = ((const Unaligned<2>*)from_a)->v;
            if (k + 1 < left) from_a += step_a;
            if constexpr (kTwo) {
                b[k] = ((const Unaligned<2>*)from_b)->v;
                if (k + 1 < left) from_b += step_b;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    // f(a's vector, b's) of each, from pixel `kFirst` of the batch on
    template <int kFirst = 0, typename Fn>
    __device__ __forceinline__ void visit(int left, Fn&& f) {
#pragma unroll
        for (int k = kFirst; k < kBatch; ++k) {
            if (k < left) f(a[k], b[kTwo ? k : 0]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // the batch that is loaded, after whose start f is called with what follows it, up to n pixels
    template <typename Fn>
    __device__ __forceinline__ void visit_all(int n, const char* from_a, int64_t step_a, const char* from_b, int64_t step_b, Fn&& f) {
        visit(n, f);
        while (n > kBatch) {
            n -= kBatch;
            from_a += kBatch * step_a;
            if constexpr (kTwo) from_b += kBatch * step_b;
            load(n, from_a, step_a, from_b, step_b);
            visit(n, f);
        }
    }
};

// The mean and centred sum of parts {mean, centred sum} of n values each, the lane's as sums about the first of them (a lane
// that has none: any part, of no values).
struct GnMerge {
    float about, values, first = 0.0f, second;
    __device__ __forceinline__ GnMerge(float2 part, float n) : about(part.x), values(n), second(n > 0.0f ? part.y : 0.0f) {}
    __device__ __forceinline__ void add(float2 part, float n) {
        const float d = part.x - about;
        values += n;
        first = __builtin_fmaf(d, n, first);
        second += __builtin_fmaf(d * d, n, n > 0.0f ? part.y : 0.0f);
    }
    // of all `all` values, over the team; ref: the same mean of a part in every lane
    __device__ __forceinline__ float2 finish(float all, float ref, int team) const {
        const float f = values > 0.0f ? first * __builtin_amdgcn_rcpf(values) : 0.0f;
        const float own = __builtin_fmaf(-first, f, second);  // (negative by rounding where there is no spread; NaN stays)
        const float d = (about - ref) + f, mean = team_sum(values * d, team) * __builtin_amdgcn_rcpf(all), t = d - mean;
        return float2{ref + mean, team_sum(__builtin_fmaf(values * t, t, own < 0.0f ? 0.0f : own), team)};
    }
};

// Where the first pass leaves a chunk's part of a group: those that a team of the second one merges lie in a run ([1, 16384,
// 320] fp16 13.4 us; a group's width apart 17.7).
__device__ __forceinline__ float2* gn_part(const GnParams& p, int image, int group, int chunk) {
    return (float2*)p.partial + ((int64_t)image * p.groups + group) * p.chunks + chunk;
}

template <typename T>
__global__ __launch_bounds__(kMaxThreads) void gn_stats_kernel(GnParams p) {
    using V = GnVec<T>;
    constexpr int kV = V::kV;
    extern __shared__ __attribute__((aligned(16))) float2 parts[];  // [rows][channels] {mean, sum of squares about it}
    const int column = (int)blockIdx.x % p.columns, chunk = (int)blockIdx.x / p.columns;
    const int image = column / p.slabs;
    const GnSlab slab = slab_of(p, column % p.slabs);
    const int64_t first = (int64_t)chunk * p.chunk_pixels;
    const int count = (int)(p.pixels - first < p.chunk_pixels ? p.pixels - first : p.chunk_pixels);
    const GnPlace at = place_of<kV>(p, slab);
    const int rows = min(p.rows_at_once, count);
    if (at.r < rows) {
        const int64_t step = p.ld_x * p.rows_at_once * (int64_t)sizeof(T);
        const char* x = (const char*)p.x + ((image * p.pixels + first + at.r) * p.ld_x + slab.c0 + at.c0) * (int64_t)sizeof(T);
        const int n = share_of(count, at.r, p.rows_at_once);
        constexpr int kBatch = 8;
        GnBatch<kBatch, false> batch;
        batch.load(n, x, step, nullptr, 0);
        float pivot[kV], s[kV] = {}, q[kV] = {};
        V::unpack(batch.a[0], pivot);
        auto add = [&](u32x4 d, u32x4) __attribute__((always_inline)) {
            float v[kV];
            V::unpack(d, v);
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                const float t = v[e] - pivot[e];
                s[e] += t;
                q[e] = __builtin_fmaf(t, t, q[e]);
            }
        };
        batch.template visit<1>(n, add);
        float seen = (float)min(n, kBatch), over = __builtin_amdgcn_rcpf(seen);
        float mean[kV], squares[kV];  // mean: from the pivot on; squares: about the mean
#pragma unroll
        for (int e = 0; e < kV; ++e) {
            mean[e] = s[e] * over;
            squares[e] = __builtin_fmaf(-s[e], mean[e], q[e]);
        }
        for (int left = n - kBatch; left > 0; left -= kBatch) {
            x += kBatch * step;
            batch.load(left, x, step, nullptr, 0);
            float off[kV];  // of the pivot from the mean
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                const float to = pivot[e] + mean[e];
                off[e] = (pivot[e] - to) + mean[e];
                pivot[e] = to;
                s[e] = q[e] = 0.0f;
            }
            batch.visit(left, add);
            const float before = seen;
            seen += (float)min(left, kBatch);
            over = __builtin_amdgcn_rcpf(seen);
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                const float sum = __builtin_fmaf(before, off[e], s[e]);
                mean[e] = sum * over;
                squares[e] += __builtin_fmaf(-sum, mean[e], __builtin_fmaf(before * off[e], off[e], q[e]));
            }
        }
        float2* to = parts + at.r * slab.channels + at.c0;
#pragma unroll
        for (int e = 0; e < kV; ++e)
            if (e >= at.skip) to[e] = float2{pivot[e] + mean[e], squares[e] < 0.0f ? 0.0f : squares[e]};
    }
    __syncthreads();
    const int teams = (int)blockDim.x / p.team, lane = (int)threadIdx.x % p.team;
    const float over_channels = 1.0f / (float)p.group_channels;
    // pixels of a row of the rows at a time: the first `longer` have one more
    const int each = count / p.rows_at_once, longer = count - each * p.rows_at_once;
    for (int g = (int)threadIdx.x / p.team; g < slab.groups; g += teams) {
        const float2* from = parts + g * p.group_channels;
        const int all = rows * p.group_channels;
        auto row_of = [&](int e) { return (int)(((float)e + 0.5f) * over_channels); };  // (e < 2^13: exact)
        auto part = [&](int e, int r) { return from[r * slab.channels + e - r * p.group_channels]; };
        auto values = [&](int r) { return (float)(r < longer ? each + 1 : each); };
        const int e0 = min(lane, all - 1), r0 = row_of(e0);
        GnMerge merge(part(e0, r0), lane < all ? values(r0) : 0.0f);
#pragma unroll 4
        for (int e = lane + p.team; e < all; e += p.team) {
            const int r = row_of(e);
            merge.add(part(e, r), values(r));
        }
        const float2 m = merge.finish((float)count * (float)p.group_channels, from[0].x, p.team);
        if (lane == 0) *gn_part(p, image, slab.g0 + g, chunk) = m;
    }
}

// mean and rstd of `groups` groups of an image from g0 on, from its chunks (in one order, whoever merges)
constexpr int kMergeTeam = 16;
__device__ __forceinline__ void merge_stats(const GnParams& p, int image, int g0, int groups, bool keep, float2* stats) {
    const int teams = (int)blockDim.x / kMergeTeam, lane = (int)threadIdx.x % kMergeTeam;
    const float values = (float)p.pixels * (float)p.group_channels;
    const float whole = (float)p.chunk_pixels * (float)p.group_channels;
    const float last = (float)(p.pixels - (p.chunks - 1) * p.chunk_pixels) * (float)p.group_channels;
    for (int g = (int)threadIdx.x / kMergeTeam; g < groups; g += teams) {
        const float2* from = gn_part(p, image, g0 + g, 0);
        const float2 own = from[min(lane, p.chunks - 1)];
        auto of = [&](int k) { return k < p.chunks - 1 ? whole : k == p.chunks - 1 ? last : 0.0f; };
        GnMerge merge(own, 0.0f);
        if (p.chunks <= kMergeTeam) merge = GnMerge(own, of(lane));
        else
            for (int k = lane; k < p.chunks; k += 4 * kMergeTeam) {
                float2 part[4];  // on their way together, past the last part that one again, of no values
#pragma unroll
                for (int i = 0; i < 4; ++i) part[i] = from[min(k + i * kMergeTeam, p.chunks - 1)];
#pragma unroll
                for (int i = 0; i < 4; ++i) merge.add(part[i], of(k + i * kMergeTeam));
            }
        const float2 m = merge.finish(values, from[0].x, kMergeTeam);
        if (lane == 0) {
            const float2 s{m.x, 1.0f / __builtin_sqrtf(m.y / values + p.eps)};
            stats[g] = s;
            if (keep) ((float2*)p.stats_out)[(int64_t)image * p.groups + g0 + g] = s;
        }
    }
    __syncthreads();
}

template <typename T>
__device__ __forceinline__ void load_channels(const void* from, int c0, float (&v)[GnVec<T>::kV]) {
    GnVec<T>::unpack(GnVec<T>::load((const char*)from + c0 * (int64_t)sizeof(T)), v);
}

// z of a channel's values, (x - mean) a + beta: a value that is the mean gives beta itself. (x a + (beta - mean a) is an
// instruction less, and off by 2^-24 of mean a.)
template <typename T>
struct GnAffine {
    static constexpr int kV = GnVec<T>::kV;
    float mean[kV], a[kV], b[kV];
    // gamma and beta are in a and b
    __device__ __forceinline__ void set(int e, float2 stats) {
        mean[e] = stats.x;
        a[e] *= stats.y;
    }
    __device__ __forceinline__ float z(int e, float x) const { return __builtin_fmaf(x - mean[e], a[e], b[e]); }
};

// y, by stores that pass the caches: kept there, it costs the reads of the next call's first pass the time to write it back
// ([1, 262144, 256] fp32 156 us, 134 so; with a kernel behind that reads y, [2, 65536, 640] fp16 150 us either way, [2,
// 16384, 640] 41 and 42).
template <typename T, FfFamily kFam>
__global__ __launch_bounds__(kMaxThreads) void gn_apply_kernel(GnParams p) {
    using V = GnVec<T>;
    constexpr int kV = V::kV;
    extern __shared__ __attribute__((aligned(16))) float2 stats[];
    const int column = (int)blockIdx.x % p.columns, chunk = (int)blockIdx.x / p.columns, image = column / p.slabs;
    const GnSlab slab = slab_of(p, column % p.slabs);
    const int64_t first = (int64_t)chunk * p.apply_pixels;
    const int count = (int)(p.pixels - first < p.apply_pixels ? p.pixels - first : p.apply_pixels);
    const GnPlace at = place_of<kV>(p, slab);
    const int n = at.r < p.rows_at_once && at.r < count ? share_of(count, at.r, p.rows_at_once) : 0;
    const int64_t row = image * p.pixels + first + (n > 0 ? at.r : 0);
    const char* x = (const char*)p.x + (row * p.ld_x + slab.c0 + at.c0) * (int64_t)sizeof(T);
    const int64_t step_x = p.ld_x * p.rows_at_once * (int64_t)sizeof(T), step_y = p.ld_y * p.rows_at_once * (int64_t)sizeof(T);
    GnBatch<4, false> batch;
    batch.load(n, x, step_x, nullptr, 0);
    merge_stats(p, image, slab.g0, slab.groups, p.stats_out != nullptr && chunk == 0, stats);
    if (n <= 0) return;
    const FfAct act = ff_act(p.activation);
    GnAffine<T> affine;
    load_channels<T>(p.gamma, slab.c0 + at.c0, affine.a);
    load_channels<T>(p.beta, slab.c0 + at.c0, affine.b);
#pragma unroll
    for (int e = 0; e < kV; ++e) affine.set(e, stats[group_of(p, at.c0 + e)]);
    char* y = (char*)p.y + (row * p.ld_y + slab.c0 + at.c0) * (int64_t)sizeof(T);
    batch.visit_all(n, x, step_x, nullptr, 0, [&](u32x4 d, u32x4) __attribute__((always_inline)) {
        float v[kV];
        V::unpack(d, v);
#pragma unroll
        for (int e = 0; e < kV; ++e) v[e] = gn_value<T, kFam>(act, affine.z(e, v[e]));
        // (in place, the vector that a row's last one overlaps may be written before this one is read: what they share is its)
        if (at.skip == 0) {
            V::store_through(y, V::pack(v));
        } else {
#pragma unroll
            for (int e = 0; e < kV; ++e)
                if (e >= at.skip) ((T*)y)[e] = (T)v[e];
        }
        y += step_y;
    });
}

// Codes by row. The row's lanes keep their channels' constants, of z as sdxl_group_norm forms it. (x a + (beta - mean a) is
// off by 2^-24 of mean a: up to 0.03 for x = 1000 throughout and eps 1e-6, where z is beta.) Every workgroup merges the parts of all groups, so that eight waves
// with a row each and a workgroup a CU beat four and two ([1, 16384, 320] fp16, both passes: 15.7 us and 18.0; [2, 1024,
// 1280] 10.4 and 11.1; sixteen 15.1 and, out of registers, 29.2).
template <typename T, FfFamily kFam, int kWaves, int kVecs>
__global__ __launch_bounds__(kWaves == 1 ? 512 : 256) void gn_rows_kernel(GnParams p) {
    extern __shared__ __attribute__((aligned(16))) float2 stats[];
    __shared__ float part[4];
    const int task = (int)blockIdx.x;
    const int image = task / p.apply_chunks, chunk = task % p.apply_chunks;
    constexpr int kRows = kWaves == 1 ? 8 : 1;  // of a workgroup at a time
    const I8Row<kWaves, kVecs> row(p.channels);
    const int64_t first = (int64_t)chunk * p.apply_pixels;
    const int count = (int)(p.pixels - first < p.apply_pixels ? p.pixels - first : p.apply_pixels);
    u32x4 d[kVecs];
    // (lanes past the row's end: its last vector; past the last row: that one)
    auto fetch = [&](int r) __attribute__((always_inline)) {
        const char* x = (const char*)p.x + (image * p.pixels + first + min(r, count - 1)) * p.ld_x * 2;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) d[i] = GnVec<T>::load(x + row.column(i) * 2);
    };
    int r = (int)threadIdx.x / (64 * kWaves);
    fetch(r);
    merge_stats(p, image, 0, p.groups, p.stats_out != nullptr && chunk == 0, stats);
    GnAffine<T> affine[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        load_channels<T>(p.gamma, row.column(i), affine[i].a);
        load_channels<T>(p.beta, row.column(i), affine[i].b);
    }
    const FfAct act = ff_act(p.activation);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) affine[i].set(e, stats[group_of(p, row.column(i) + e)]);
    }
    for (; r < count; r += kRows) {
        float v[kVecs][8];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            GnVec<T>::unpack(d[i], v[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = ff_value<kFam>(act, affine[i].z(e, v[i][e]));
        }
        fetch(r + kRows);
        const int64_t at = image * p.pixels + first + r;
        const float scale = row.quantise(v, part, p.q + at * p.ld_q, 0);
        if (row.lane == 0) p.q_scale[at] = scale;
    }
}

// The thread's constants of the gradients: z = (x - mean) a + beta.
template <typename T>
struct GnBackward {
    static constexpr int kV = GnVec<T>::kV;
    float mean[kV], rstd[kV], a[kV], beta[kV];
    __device__ __forceinline__ void load(const GnParams& p, int image, int c0) {
        load_channels<T>(p.gamma, c0, a);
        load_channels<T>(p.beta, c0, beta);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
            const float2 s = ((const float2*)p.stats)[(int64_t)image * p.groups + group_of(p, c0 + e)];
            mean[e] = s.x;
            rstd[e] = s.y;
            a[e] *= s.y;
        }
    }
};

// The sums of dz and of dz n by channel, and of both by group with gamma.
template <typename T, FfFamily kFam>
__global__ __launch_bounds__(kMaxThreads) void gn_sums_kernel(GnParams p) {
    using V = GnVec<T>;
    constexpr int kV = V::kV;
    extern __shared__ __attribute__((aligned(16))) float2 parts[];  // [rows][channels]
    const int column = (int)blockIdx.x % p.columns, chunk = (int)blockIdx.x / p.columns;
    const int image = column / p.slabs, task = image * p.chunks + chunk;
    const GnSlab slab = slab_of(p, column % p.slabs);
    const int64_t first = (int64_t)chunk * p.chunk_pixels;
    const int count = (int)(p.pixels - first < p.chunk_pixels ? p.pixels - first : p.chunk_pixels);
    const GnPlace at = place_of<kV>(p, slab);
    const int rows = min(p.rows_at_once, count);
    if (at.r < rows) {
        const int64_t row = image * p.pixels + first + at.r;
        const char* x = (const char*)p.x + (row * p.ld_x + slab.c0 + at.c0) * (int64_t)sizeof(T);
        const char* dy = (const char*)p.dy + (row * p.ld_dy + slab.c0 + at.c0) * (int64_t)sizeof(T);
        const int64_t step_x = p.ld_x * p.rows_at_once * (int64_t)sizeof(T), step_dy = p.ld_dy * p.rows_at_once * (int64_t)sizeof(T);
        const int n = share_of(count, at.r, p.rows_at_once);
        GnBatch<4, true> batch;
        batch.load(n, x, step_x, dy, step_dy);
        const FfAct act = ff_act(p.activation);
        GnBackward<T> b;
        b.load(p, image, slab.c0 + at.c0);
        float s1[kV] = {}, s2[kV] = {};
        auto add = [&](u32x4 dx, u32x4 dd) __attribute__((always_inline)) {
            float v[kV], d[kV];
            V::unpack(dx, v);
            V::unpack(dd, d);
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                const float t = v[e] - b.mean[e];
                const float dz = kFam == kFamLinear && p.activation == SDXL_ACT_NONE ? d[e] : d[e] * gn_slope<T, kFam>(act, __builtin_fmaf(t, b.a[e], b.beta[e]));
                s1[e] += dz;
                s2[e] = __builtin_fmaf(dz, t, s2[e]);
            }
        };
        batch.visit_all(n, x, step_x, dy, step_dy, add);
        float2* to = parts + at.r * slab.channels + at.c0;
#pragma unroll
        for (int e = 0; e < kV; ++e)
            if (e >= at.skip) to[e] = float2{s1[e], s2[e] * b.rstd[e]};
    }
    __syncthreads();
    for (int c = threadIdx.x; c < slab.channels; c += blockDim.x) {
        float2 sum = parts[c];
#pragma unroll 4
        for (int r = 1; r < rows; ++r) {
            sum.x += parts[r * slab.channels + c].x;
            sum.y += parts[r * slab.channels + c].y;
        }
        ((float2*)p.channel_sums)[(int64_t)task * p.channels + slab.c0 + c] = sum;
        const float gamma = (float)((const T*)p.gamma)[slab.c0 + c];
        parts[c] = float2{sum.x * gamma, sum.y * gamma};  // (this thread's column alone)
    }
    __syncthreads();
    const int teams = (int)blockDim.x / p.team, lane = (int)threadIdx.x % p.team;
    for (int g = (int)threadIdx.x / p.team; g < slab.groups; g += teams) {
        float a = 0.0f, b = 0.0f;
        for (int c = lane; c < p.group_channels; c += p.team) {
            a += parts[g * p.group_channels + c].x;
            b += parts[g * p.group_channels + c].y;
        }
        a = team_sum(a, p.team);
        b = team_sum(b, p.team);
        if (lane == 0) *gn_part(p, image, slab.g0 + g, chunk) = float2{a, b};
    }
}

constexpr int kParamChannels = 32;  // of a workgroup that adds up dgamma and dbeta

// dx, and in workgroups of their own, the last ones (in front they push dx's off their data's XCDs: [8, 1024, 1280] 27.1 us and
// 24.4), dgamma and dbeta.
template <typename T, FfFamily kFam>
__global__ __launch_bounds__(kMaxThreads) void gn_dx_kernel(GnParams p) {
    using V = GnVec<T>;
    constexpr int kV = V::kV;
    extern __shared__ __attribute__((aligned(16))) float2 means[];
    const int tasks = p.y != nullptr ? p.apply_chunks * p.columns : 0, task = (int)blockIdx.x;
    if (task >= tasks) {
        const int c = (task - tasks) * kParamChannels + (int)threadIdx.x % kParamChannels;
        const int lanes = (int)blockDim.x / kParamChannels, lane = (int)threadIdx.x / kParamChannels, parts = p.batch * p.chunks;
        double2* const joined = (double2*)means;
        double2 sum{0.0, 0.0};  // (in 64 bits: a lane may have thousands of images' parts)
        if (c < p.channels)
#pragma unroll 8
            for (int k = lane; k < parts; k += lanes) {
                const float2 a = ((const float2*)p.channel_sums)[(int64_t)k * p.channels + c];
                sum.x += (double)a.x;
                sum.y += (double)a.y;
            }
        joined[threadIdx.x] = sum;
        __syncthreads();
        if (lane == 0 && c < p.channels) {
            for (int k = 1; k < lanes; ++k) {
                sum.x += joined[k * kParamChannels + threadIdx.x].x;
                sum.y += joined[k * kParamChannels + threadIdx.x].y;
            }
            if (p.dbeta != nullptr) ((T*)p.dbeta)[c] = (T)(float)sum.x;
            if (p.dgamma != nullptr) ((T*)p.dgamma)[c] = (T)(float)sum.y;
        }
        return;
    }
    const int column = task % p.columns, chunk = task / p.columns, image = column / p.slabs;
    const GnSlab slab = slab_of(p, column % p.slabs);
    const int64_t first = (int64_t)chunk * p.apply_pixels;
    const int count = (int)(p.pixels - first < p.apply_pixels ? p.pixels - first : p.apply_pixels);
    const GnPlace at = place_of<kV>(p, slab);
    const int n = at.r < p.rows_at_once && at.r < count ? share_of(count, at.r, p.rows_at_once) : 0;
    const int64_t row = image * p.pixels + first + (n > 0 ? at.r : 0);
    const char* x = (const char*)p.x + (row * p.ld_x + slab.c0 + at.c0) * (int64_t)sizeof(T);
    const char* dy = (const char*)p.dy + (row * p.ld_dy + slab.c0 + at.c0) * (int64_t)sizeof(T);
    const int64_t step_x = p.ld_x * p.rows_at_once * (int64_t)sizeof(T), step_dy = p.ld_dy * p.rows_at_once * (int64_t)sizeof(T);
    const int64_t step_dx = p.ld_y * p.rows_at_once * (int64_t)sizeof(T);
    GnBatch<4, true> batch;
    batch.load(n, x, step_x, dy, step_dy);
    GnBackward<T> b;  // (on the way before the merge)
    b.load(p, image, slab.c0 + at.c0);
    const int teams = (int)blockDim.x / p.team, lane = (int)threadIdx.x % p.team;
    const float over = 1.0f / ((float)p.pixels * (float)p.group_channels);
    for (int g = (int)threadIdx.x / p.team; g < slab.groups; g += teams) {
        const float2* from = gn_part(p, image, slab.g0 + g, 0);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
        for (int k = lane; k < p.chunks; k += p.team) {
            s1 += from[k].x;
            s2 += from[k].y;
        }
        s1 = team_sum(s1, p.team);
        s2 = team_sum(s2, p.team);
        if (lane == 0) means[g] = float2{s1 * over, s2 * over};
    }
    __syncthreads();
    if (n <= 0) return;
    const FfAct act = ff_act(p.activation);
    float a1[kV], a2[kV];  // dx = a dz - a1 - (x - mean) a2
#pragma unroll
    for (int e = 0; e < kV; ++e) {
        const float2 m = means[group_of(p, at.c0 + e)];
        a1[e] = b.rstd[e] * m.x;
        a2[e] = b.rstd[e] * b.rstd[e] * m.y;
    }
    char* dx = (char*)p.y + (row * p.ld_y + slab.c0 + at.c0) * (int64_t)sizeof(T);
    batch.visit_all(n, x, step_x, dy, step_dy, [&](u32x4 xd, u32x4 dd) __attribute__((always_inline)) {
        float v[kV], d[kV];
        V::unpack(xd, v);
        V::unpack(dd, d);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
            const float t = v[e] - b.mean[e];
            const float dz = kFam == kFamLinear && p.activation == SDXL_ACT_NONE ? d[e] : d[e] * gn_slope<T, kFam>(act, __builtin_fmaf(t, b.a[e], b.beta[e]));
            v[e] = __builtin_fmaf(-t, a2[e], __builtin_fmaf(dz, b.a[e], -a1[e]));
        }
        V::store_through(dx, V::pack(v));
        dx += step_dx;
    });
}

// ---- One launch, where a set of groups of an image fits a workgroup's registers, eight vectors a thread: [2, 256, 1280] fp16
// 6.1 us on the device (two passes 9.0), [2, 576, 1280] 8.2 (9.6); with twelve, [2, 1024, 1280], 9.4 (9.2). (The gradients so:
// their sets are a workgroup's for all images, whose arithmetic is too much for it; [2, 256, 1280] 14.5, two passes 11.4.)

constexpr int kHeldVecs = 32;  // vectors of a set's row at most

// Sums by group over the workgroup, of what its threads have of the two groups that a vector may lie in.
struct GnHeld {
    int vecs, rows;
    float2 *parts, *totals;  // [vecs][rows], [vecs]
    int* group;              // [vecs]: a vector's first group

    __device__ __forceinline__ GnHeld(const GnParams& p, char* lds, const GnPlace& at) : vecs(p.vecs), rows(p.rows_at_once), parts((float2*)lds) {
        totals = parts + vecs * rows;
        group = (int*)(totals + vecs);
        if (at.r == 0) group[(int)threadIdx.x] = group_of(p, at.c0);  // (read behind the first barrier)
    }
    static size_t bytes(const GnParams& p) { return (size_t)p.vecs * (p.rows_at_once + 1) * 8 + (size_t)p.vecs * 4; }

    // x: of vector v's first group, y: of the next one; returns both groups' sums
    __device__ __forceinline__ float2 sums(const GnPlace& at, int v, float2 mine) const {
        if (at.r < rows) parts[v * rows + at.r] = mine;
        __syncthreads();
        const int lane = threadIdx.x & 63;
        for (int w = (int)threadIdx.x >> 6; w < vecs; w += (int)blockDim.x >> 6) {
            float2 t{0.0f, 0.0f};
            for (int r = lane; r < rows; r += 64) {
                t.x += parts[w * rows + r].x;
                t.y += parts[w * rows + r].y;
            }
            t.x = reduce64(t.x, Add{});
            t.y = reduce64(t.y, Add{});
            if (lane == 0) totals[w] = t;
        }
        __syncthreads();
        const int g = group[v];
        float2 all{0.0f, 0.0f};
        for (int w = 0; w < vecs; ++w) {
            const int d = group[w] - g;
            const float2 t = totals[w];
            all.x += d == 0 ? t.x : d == -1 ? t.y : 0.0f;
            all.y += d == 0 ? t.y : d == 1 ? t.x : 0.0f;
        }
        return all;
    }
};

// The workgroup's image and set: neighbouring sets, which share cache lines, on one XCD.
__device__ __forceinline__ int held_task() {
    const int n = (int)gridDim.x, id = (int)blockIdx.x, xcd = id & 7, per = n >> 3, extra = n & 7;
    return xcd * per + (xcd < extra ? xcd : extra) + (id >> 3);
}

// Two passes over the registers: the mean from sums about a value of the group, then the squares about the mean.
template <typename T, FfFamily kFam, int kHold>
__global__ __launch_bounds__(kMaxThreads) void gn_held_kernel(GnParams p) {
    using V = GnVec<T>;
    constexpr int kV = V::kV;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int task = held_task(), image = task / p.slabs;
    const GnSlab slab = slab_of(p, task % p.slabs);
    const GnPlace at = place_of<kV>(p, slab);
    const int pixels = (int)p.pixels, n = at.r < p.rows_at_once && at.r < pixels ? share_of(pixels, at.r, p.rows_at_once) : 0;
    const int64_t row = image * p.pixels + (n > 0 ? at.r : 0);
    const char* x = (const char*)p.x + (row * p.ld_x + slab.c0 + at.c0) * (int64_t)sizeof(T);
    GnBatch<kHold, false> batch;
    batch.load(n, x, p.ld_x * p.rows_at_once * (int64_t)sizeof(T), nullptr, 0);
    const int g = group_of(p, at.c0), next = (g + 1) * p.group_channels - at.c0;  // elements from `next` on: the next group's
    const int g2 = min(g + 1, slab.groups - 1);
    const T* pivots = (const T*)p.x + image * p.pixels * p.ld_x + slab.c0;
    const float2 pivot{(float)pivots[g * p.group_channels], (float)pivots[g2 * p.group_channels]};
    GnAffine<T> affine;
    load_channels<T>(p.gamma, slab.c0 + at.c0, affine.a);
    load_channels<T>(p.beta, slab.c0 + at.c0, affine.b);
    const GnHeld held(p, lds, at);
    const int v = (int)threadIdx.x % p.vecs;
    auto split = [&](const float (&s)[kV]) __attribute__((always_inline)) {
        float2 sum{0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < kV; ++e) {
            const float t = e >= at.skip ? s[e] : 0.0f;
            if (e < next) sum.x += t;
            else sum.y += t;
        }
        return sum;
    };
    const float over = 1.0f / ((float)pixels * (float)p.group_channels);
    float s[kV] = {};
    batch.visit(n, [&](u32x4 d, u32x4) __attribute__((always_inline)) {
        float u[kV];
        V::unpack(d, u);
#pragma unroll
        for (int e = 0; e < kV; ++e) s[e] += u[e] - (e < next ? pivot.x : pivot.y);
    });
    const float2 first = held.sums(at, v, split(s));
    const float2 mean{__builtin_fmaf(first.x, over, pivot.x), __builtin_fmaf(first.y, over, pivot.y)};
#pragma unroll
    for (int e = 0; e < kV; ++e) s[e] = 0.0f;
    batch.visit(n, [&](u32x4 d, u32x4) __attribute__((always_inline)) {
        float u[kV];
        V::unpack(d, u);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
            const float t = u[e] - (e < next ? mean.x : mean.y);
            s[e] = __builtin_fmaf(t, t, s[e]);
        }
    });
    const float2 second = held.sums(at, v, split(s));
    const float2 stats{mean.x, 1.0f / __builtin_sqrtf(__builtin_fmaf(second.x, over, p.eps))};
    const float2 stats2{mean.y, 1.0f / __builtin_sqrtf(__builtin_fmaf(second.y, over, p.eps))};
    if (n <= 0) return;
    if (p.stats_out != nullptr && at.r == 0) {  // the threads that have a group's first channel
        float2* to = (float2*)p.stats_out + (int64_t)image * p.groups + slab.g0;
        if (at.c0 == g * p.group_channels) to[g] = stats;
        if (next < kV) to[g + 1] = stats2;
    }
    const FfAct act = ff_act(p.activation);
#pragma unroll
    for (int e = 0; e < kV; ++e) affine.set(e, e < next ? stats : stats2);
    char* y = (char*)p.y + (row * p.ld_y + slab.c0 + at.c0) * (int64_t)sizeof(T);
    const int64_t step_y = p.ld_y * p.rows_at_once * (int64_t)sizeof(T);
    batch.visit(n, [&](u32x4 d, u32x4) __attribute__((always_inline)) {
        float u[kV];
        V::unpack(d, u);
#pragma unroll
        for (int e = 0; e < kV; ++e) u[e] = gn_value<T, kFam>(act, affine.z(e, u[e]));
        V::store(y, V::pack(u));
        y += step_y;
    });
}

// ---- launches

int elem_of(GnType type) { return type == kGnF32 ? 4 : 2; }

// Groups of a slab: the smallest divisor of the groups that makes `least` bytes of a row (and whole vectors), else all.
constexpr int64_t kSlabBytes = 512, kHeldBytes = 64;
int slab_groups_of(const GnParams& p, GnType type, int64_t least) {
    const int64_t bytes = (int64_t)p.group_channels * elem_of(type);
    for (int d = (int)((least + bytes - 1) / bytes); d < p.groups; ++d)
        if (p.groups % d == 0 && (d * bytes % 16 == 0 || least == kSlabBytes)) return d;
    return p.groups;
}
int64_t vecs_of(const GnParams& p, GnType type, int slab_groups) {
    return ((int64_t)p.group_channels * slab_groups * elem_of(type) + 15) / 16;
}

constexpr int64_t kMaxColumns = 1 << 22;  // of kMaxThreads threads each: below 2^32

// Threads of a workgroup: of 4 to 8 waves the most whose lanes have work, the most of equals.
int threads_of(int vecs) {
    int best = 0, best_used = -1;
    for (int t = 256; t <= kMaxThreads; t += 64) {
        const int used = t / vecs * vecs * 1024 / t;
        if (t >= vecs && used >= best_used) {
            best = t;
            best_used = used;
        }
    }
    return best;
}

int team_of(int groups, int threads) { return 64 * groups <= threads ? 64 : 16; }

// Workgroups of the two passes, and the rounds that a chunk has a multiple of. One workgroup a CU
// reads fast enough and leaves few parts: [2, 16384, 640] fp16 25.9 us with 256 and 512, 26.4 with 512 and 512, 29.5 with 256
// and 256, 25.1 with 256 and 768; [1, 16384, 320] 13.4, 16.8, 14.1, 13.4.
constexpr int kFirstTasks = 256, kSecondTasks = 512;
constexpr int kBatchRounds = 4;

// `columns` (images by slabs) in chunks of whole rounds of `rows` pixels: `tasks` chunks in all or a little fewer, of
// whole batches of rounds; more where a chunk would have over 1024 (what a thread adds up).
int64_t chunk_of(int64_t columns, int64_t pixels, int rows, int tasks, int batch) {
    const int64_t each = tasks / columns < 1 ? 1 : tasks / columns;
    const int64_t rounds = (pixels + rows - 1) / rows, chunk = ((rounds + each - 1) / each + batch - 1) / batch * batch;
    return (chunk < 1024 ? chunk : 1024) * rows;
}

template <typename T, typename Fn>
hipError_t by_family(int32_t activation, Fn&& f) {
    switch (activation) {
    case SDXL_ACT_NONE:
    case SDXL_ACT_RELU: return f.template operator()<T, kFamLinear>();
    case SDXL_ACT_GELU: return f.template operator()<T, kFamErf>();
    case SDXL_ACT_GELU_TANH: return f.template operator()<T, kFamTanh>();
    default: return f.template operator()<T, kFamSigmoid>();
    }
}

template <typename Fn>
hipError_t by_type(GnType type, int32_t activation, Fn&& f) {
    return type == kGnF16 ? by_family<_Float16>(activation, f) : type == kGnBf16 ? by_family<__bf16>(activation, f) : by_family<float>(activation, f);
}

// Fills in what the kernels of `threads` threads need.
void lay_out(GnParams& p, GnType type, int slab_groups, int threads) {
    p.slab_groups = slab_groups;
    p.slabs = p.groups / p.slab_groups;
    p.vecs = (int32_t)vecs_of(p, type, p.slab_groups);
    p.rows_at_once = threads / p.vecs;
    p.team = team_of(p.slab_groups, threads);
    p.columns = p.batch * p.slabs;
}

void cut_second(GnParams& p, int64_t columns, int rows, int tasks, int batch) {
    p.apply_pixels = chunk_of(columns, p.pixels, rows, tasks, batch);
    p.apply_chunks = (int32_t)((p.pixels + p.apply_pixels - 1) / p.apply_pixels);
}

// Codes: a wave a row up to 5 vectors a lane, else four.
constexpr int kRowVecs = 5;

template <typename T, FfFamily kFam, int kWaves>
hipError_t launch_rows_of(const GnParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)(p.batch * p.apply_chunks)), block(kWaves == 1 ? 512 : 256);
    const size_t lds = (size_t)p.groups * 8;
    switch ((p.vecs + 64 * kWaves - 1) / (64 * kWaves)) {
    case 1: hipLaunchKernelGGL((gn_rows_kernel<T, kFam, kWaves, 1>), grid, block, lds, stream, p); break;
    case 2: hipLaunchKernelGGL((gn_rows_kernel<T, kFam, kWaves, 2>), grid, block, lds, stream, p); break;
    case 3: hipLaunchKernelGGL((gn_rows_kernel<T, kFam, kWaves, 3>), grid, block, lds, stream, p); break;
    case 4: hipLaunchKernelGGL((gn_rows_kernel<T, kFam, kWaves, 4>), grid, block, lds, stream, p); break;
    case 5: hipLaunchKernelGGL((gn_rows_kernel<T, kFam, kWaves, 5>), grid, block, lds, stream, p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_rows(const GnParams& params, GnType type, hipStream_t stream) {
    GnParams p = params;
    p.vecs = (p.channels + 7) / 8;
    const bool wave = p.vecs <= 64 * kRowVecs;
    cut_second(p, p.batch, wave ? 8 : 1, wave ? 256 : 512, 1);
    auto launch = [&]<typename T, FfFamily kFam>() {
        return wave ? launch_rows_of<T, kFam, 1>(p, stream) : launch_rows_of<T, kFam, 4>(p, stream);
    };
    return type == kGnF16 ? by_family<_Float16>(p.activation, launch) : by_family<__bf16>(p.activation, launch);
}

}  // namespace

namespace {

// The vectors that a thread of the held kernels has, 0 where they do not take the call: a set of groups that they can tell
// apart (a vector lies in two at most) and hold.
constexpr int kHolds[] = {1, 2, 4, 8};
int hold_of(const GnParams& p, GnType type, int& slab_groups, int& threads) {
    const int kV = 16 / elem_of(type);
    slab_groups = slab_groups_of(p, type, kHeldBytes);
    const int64_t vecs = vecs_of(p, type, slab_groups);
    if (slab_groups > 1 && p.group_channels < kV && (p.group_channels * 2 != kV || slab_groups * p.group_channels % kV != 0)) return 0;
    if (vecs > kHeldVecs || p.pixels > (1 << 16) || (int64_t)p.batch * (p.groups / slab_groups) > kMaxColumns) return 0;
    threads = (int)(vecs * p.pixels < kMaxThreads ? (vecs * p.pixels + 63) / 64 * 64 : kMaxThreads);
    const int rows = threads / (int)vecs, needed = (int)((p.pixels + rows - 1) / rows);
    for (int hold : kHolds)
        if (hold >= needed) return hold;
    return 0;
}

bool fast_of(const GnParams& p, GnType type) {
    const int slab_groups = slab_groups_of(p, type, kSlabBytes);
    const int64_t vecs = vecs_of(p, type, slab_groups), columns = (int64_t)p.batch * (p.groups / slab_groups);
    return p.batch > 0 && p.pixels > 0 && p.channels >= 16 / elem_of(type) && vecs <= kMaxThreads && columns <= kMaxColumns &&
           p.groups <= 4096 && p.pixels < (1 << 28) && p.ld_x <= (1 << 20) && p.ld_y <= (1 << 20) && p.ld_dy <= (1 << 20);
}

}  // namespace

GnPlan gn_plan(const GnParams& p, GnType type, GnCall call) {
    if (!fast_of(p, type) || (call == kGnRows && p.channels > 4 * 64 * 8 * kRowVecs)) return {false, 0, 1, p.pixels};
    int slab_groups, threads;
    if (call == kGnForward) {
        const int hold = hold_of(p, type, slab_groups, threads);
        if (hold > 0) return {true, hold, 0, 0};
    }
    slab_groups = slab_groups_of(p, type, kSlabBytes);
    const int vecs = (int)vecs_of(p, type, slab_groups);
    const int64_t columns = (int64_t)p.batch * (p.groups / slab_groups);
    const int rows = threads_of(vecs) / vecs;
    auto chunks_of = [&](int64_t chunk) { return (p.pixels + chunk - 1) / chunk; };
    int64_t chunk = chunk_of(columns, p.pixels, rows, kFirstTasks, kBatchRounds);
    // The gradients' first pass of 16-bit types, whose slopes keep the vector units busy, takes two workgroups a CU where an
    // image's parts stay few for it and they come out even: [2, 65536, 640] 162 us (one a CU 175), [2, 16384, 640] 42.8 (46.7), [8,
    // 1024, 1280] 24.7 (25.8), [2, 4096, 640] 16.7 (17.6). Three columns, which keep one, would gain or stay: [3, 9216, 320] 26.3
    // (28.3), [3, 4096, 320] 17.0 (17.7), [3, 16384, 320] 43.7 both. Else: of one column [1, 16384, 320] 23.3 (19.2), of two [2, 131072,
    // 256] 113.8 (112.7); uneven [2, 6144, 960] 27.6 (25.4); fp32 [4, 4096, 320] 20.5 (19.3).
    if (call == kGnBackward && type != kGnF32 && columns >= 4) {
        auto rounds_of = [&](int64_t c) { return (columns * chunks_of(c) + kFirstTasks - 1) / kFirstTasks * c; };
        const int64_t half = chunk_of(columns, p.pixels, rows, 2 * kFirstTasks, kBatchRounds);
        if (rounds_of(half) <= rounds_of(chunk)) chunk = half;
    }
    return {true, 0, (int32_t)chunks_of(chunk), chunk};
}

namespace {

template <typename T, FfFamily kFam, int kHold>
hipError_t launch_held_of(const GnParams& p, int threads, hipStream_t stream) {
    hipLaunchKernelGGL((gn_held_kernel<T, kFam, kHold>), dim3((unsigned)(p.batch * p.slabs)), dim3(threads), GnHeld::bytes(p), stream, p);
    return hipGetLastError();
}

hipError_t launch_held(const GnParams& params, GnType type, int hold, hipStream_t stream) {
    GnParams p = params;
    int slab_groups, threads;
    hold_of(p, type, slab_groups, threads);
    lay_out(p, type, slab_groups, threads);
    return by_type(type, p.activation, [&]<typename T, FfFamily kFam>() {
        switch (hold) {
        case 1: return launch_held_of<T, kFam, 1>(p, threads, stream);
        case 2: return launch_held_of<T, kFam, 2>(p, threads, stream);
        case 4: return launch_held_of<T, kFam, 4>(p, threads, stream);
        case 8: return launch_held_of<T, kFam, 8>(p, threads, stream);
        }
        return hipErrorInvalidValue;
    });
}

}  // namespace

hipError_t launch_gn_forward(const GnPlan& plan, const GnParams& params, GnType type, hipStream_t stream) {
    GnParams p = params;
    if (!plan.fast) {
        const hipError_t err = launch_gn_stats_general(p, type, stream);
        return err != hipSuccess ? err : launch_gn_apply_general(p, type, stream);
    }
    if (plan.hold > 0) return launch_held(p, type, plan.hold, stream);
    const int slab_groups = slab_groups_of(p, type, kSlabBytes), threads = threads_of((int)vecs_of(p, type, slab_groups));
    lay_out(p, type, slab_groups, threads);
    {
        const dim3 grid((unsigned)(p.columns * p.chunks));
        const size_t lds = (size_t)p.rows_at_once * p.slab_groups * p.group_channels * 8;
        if (type == kGnF16) hipLaunchKernelGGL(gn_stats_kernel<_Float16>, grid, dim3(threads), lds, stream, p);
        else if (type == kGnBf16) hipLaunchKernelGGL(gn_stats_kernel<__bf16>, grid, dim3(threads), lds, stream, p);
        else hipLaunchKernelGGL(gn_stats_kernel<float>, grid, dim3(threads), lds, stream, p);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    if (p.q != nullptr) return launch_rows(p, type, stream);
    cut_second(p, p.columns, p.rows_at_once, kSecondTasks, kBatchRounds);
    return by_type(type, p.activation, [&]<typename T, FfFamily kFam>() {
        hipLaunchKernelGGL((gn_apply_kernel<T, kFam>), dim3((unsigned)(p.columns * p.apply_chunks)), dim3(threads), (size_t)p.slab_groups * 8, stream, p);
        return hipGetLastError();
    });
}

hipError_t launch_gn_backward(const GnPlan& plan, const GnParams& params, GnType type, hipStream_t stream) {
    GnParams p = params;
    const bool parameters = p.dgamma != nullptr || p.dbeta != nullptr;
    if (!plan.fast) {
        hipError_t err = hipSuccess;
        if (p.batch > 0 && p.pixels > 0) {
            err = launch_gn_sums_general(p, type, stream);
            if (err == hipSuccess && p.y != nullptr) err = launch_gn_dx_general(p, type, stream);
        }
        return err == hipSuccess && parameters ? launch_gn_parameters_general(p, type, stream) : err;
    }
    const int slab_groups = slab_groups_of(p, type, kSlabBytes), threads = threads_of((int)vecs_of(p, type, slab_groups));
    lay_out(p, type, slab_groups, threads);
    const hipError_t err = by_type(type, p.activation, [&]<typename T, FfFamily kFam>() {
        hipLaunchKernelGGL((gn_sums_kernel<T, kFam>), dim3((unsigned)(p.columns * p.chunks)), dim3(threads),
                           (size_t)p.rows_at_once * p.slab_groups * p.group_channels * 8, stream, p);
        return hipGetLastError();
    });
    if (err != hipSuccess) return err;
    cut_second(p, p.columns, p.rows_at_once, kSecondTasks, kBatchRounds);
    const int64_t grid = (p.y != nullptr ? (int64_t)p.columns * p.apply_chunks : 0) + (parameters ? (p.channels + kParamChannels - 1) / kParamChannels : 0);
    const size_t lds = std::max((size_t)p.slab_groups * sizeof(float2), (size_t)threads * sizeof(double2));
    return by_type(type, p.activation, [&]<typename T, FfFamily kFam>() {
        hipLaunchKernelGGL((gn_dx_kernel<T, kFam>), dim3((unsigned)grid), dim3(threads), lds, stream, p);
        return hipGetLastError();
    });
}

}  // namespace sdxl_hip
