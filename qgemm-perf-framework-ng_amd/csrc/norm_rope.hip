// Norms of every query and key head with the position rotation, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w over the D elements of a head (w null: y = x)
//   the first R elements turn by the position's angles: for a pair (a, b)
//   a' = a cos - b sin, b' = b cos + a sin; pairs (i, i + R/2), or (2i, 2i + 1)
//
// HBM-bound: each element is read once and written once. Eight elements a lane,
// D / 8 lanes a row; the row's sum and the rotation's partners go between lanes.
// The sum of squares, the norm and the rotation are in fp32 whatever the types;
// the result is rounded once. 2047 tokens of 64 heads of 128, fp32: 24.4 us,
// 5.5 TB/s on fixed inputs (a copy of as many bytes, which the last-level cache
// holds: 6.9; of gigabytes: 4.8); 16 tokens of 40 heads 3.5 us, of which an empty
// launch is 2.1.
#include "io_types.h"
#include "kv_kernels.h"

namespace pfng {
namespace {

constexpr int kNormThreads = 256;

template <int D, class In, class Out>
__global__ __launch_bounds__(kNormThreads) void qk_norm_rope_kernel(NormRopeArgs a) {
    constexpr int kLanes = D / 8, kRows = kNormThreads / kLanes;
    const int j = threadIdx.x % kLanes;
    const int heads = a.q_heads + a.kv_heads;
    const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / kLanes;
    const bool on = row < a.tokens * heads;
    const int64_t t = on ? row / heads : 0;
    const int h = on ? int(row - t * heads) : 0;
    const bool key = h >= a.q_heads;
    const int head = key ? h - a.q_heads : h;
    const In *src = static_cast<const In *>(key ? a.k : a.q) + t * (key ? a.k_stride : a.q_stride) + int64_t(head) * D;
    f32x8 x = on ? load8(src + 8 * j) : f32x8{};
    const float *w = key ? a.k_weight : a.q_weight;
    if (w) {
        float ss = 0.0f;
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
        ss = butterfly<kLanes / 2>(ss, [](float p, float q) { return p + q; });
        const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
        const f32x8 g = *reinterpret_cast<const f32x8 *>(w + 8 * j);
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
    }
    const int half = a.rot_dim / 2, e = 8 * j;
    const int64_t position = a.rot_dim ? a.positions[t] : 0;
    const bool inside = !a.rot_dim || (position >= 0 && position < a.table_rows);
    const float *angles = a.cos_sin + (inside ? position : 0) * a.rot_dim;
    if (a.adjacent) {
        if (e < a.rot_dim) {
            const f32x4 c = *reinterpret_cast<const f32x4 *>(angles + e / 2);
            const f32x4 s = *reinterpret_cast<const f32x4 *>(angles + half + e / 2);
            for (int i = 0; i < 4; ++i) {
                const float u = x[2 * i], v = x[2 * i + 1];
                x[2 * i] = u * c[i] - v * s[i];
                x[2 * i + 1] = v * c[i] + u * s[i];
            }
        }
    } else {
        const bool low = e < half, turned = e < a.rot_dim;
        const int partner = turned ? (low ? j + half / 8 : j - half / 8) : j;
        f32x8 y;
        const int lane = threadIdx.x % 64;
        for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], lane - j + partner, 64);
        if (turned) {
            const int p = low ? e : e - half;
            const f32x8 c = *reinterpret_cast<const f32x8 *>(angles + p);
            const f32x8 s = *reinterpret_cast<const f32x8 *>(angles + half + p);
            for (int i = 0; i < 8; ++i) x[i] = low ? x[i] * c[i] - y[i] * s[i] : x[i] * c[i] + y[i] * s[i];
        }
    }
    if (!inside)
        for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
    if (!on) return;
    Out *dst = static_cast<Out *>(key ? a.k_out : a.q_out) + t * (key ? a.k_out_stride : a.q_out_stride) +
               int64_t(head) * D;
    store8(dst + 8 * j, x);
}

template <int D, class In>
hipError_t launch_out(const NormRopeArgs &a, int out_type, hipStream_t s) {
    constexpr int kRows = kNormThreads / (D / 8);
    const dim3 g((unsigned)((a.tokens * (a.q_heads + a.kv_heads) + kRows - 1) / kRows));
    switch (out_type) {
    case 0: qk_norm_rope_kernel<D, In, float><<<g, kNormThreads, 0, s>>>(a); break;
    case 1: qk_norm_rope_kernel<D, In, __bf16><<<g, kNormThreads, 0, s>>>(a); break;
    default: qk_norm_rope_kernel<D, In, _Float16><<<g, kNormThreads, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const NormRopeArgs &a, int in_type, int out_type, hipStream_t s) {
    switch (in_type) {
    case 0: return launch_out<D, float>(a, out_type, s);
    case 1: return launch_out<D, __bf16>(a, out_type, s);
    default: return launch_out<D, _Float16>(a, out_type, s);
    }
}

}  // namespace

hipError_t launch_qk_norm_rope(const NormRopeArgs &a, int in_type, int out_type, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 64: return launch_dim<64>(a, in_type, out_type, s);
    case 128: return launch_dim<128>(a, in_type, out_type, s);
    default: return launch_dim<256>(a, in_type, out_type, s);
    }
}

}  // namespace pfng
