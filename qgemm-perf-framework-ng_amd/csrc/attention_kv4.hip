// Attention over the paged 4-bit cache (format: kv_layout.h).
//
//   out[row] = sum_j softmax_j(scale * q[row] . k_j) v_j over the keys j that the row's mask leaves;
//   a row without any key is zeros
//
// One pass over the keys with a running maximum and sum (Milakov and Gimelshein's
// online softmax). The (query, head) pairs that share a key head are the rows of
// one product: 16 rows x 32 keys a wave and step, v_mfma_f32_16x16x32_f16.
//
// S^T = K Q^T: lane (g = lane / 16, n = lane % 16) ends with row n's scores of
// tokens 8g..8g+7 (the rows of the two 16-token tiles are ordered so that these
// are neighbours), which is the operand layout that O^T += V^T P^T takes for P:
// the probabilities stay in their lane.
//
// The nibbles enter the products as exact numbers and the block scales outside:
//   keys: q - 8 is exact in fp16; a block's product is added to the score times
//     the key's scale in fp32. For bf16 results the masked nibble q itself is the
//     operand, as the fp16 subnormal q 2^-24 (or 16 q 2^-24, with the query elements
//     there divided by 16), and the product starts from -8 2^-24 sum(q-row): half
//     the instructions. The matrix instruction aligns a subnormal's products as if
//     its leading bit were 2^-14, so that the sum of 32 is 7e-7 of its largest term
//     off (measured), against 1.5e-8 with q - 8: hence not for fp32 and fp16.
//   values: q - 8 is exact in fp16, and P times the block's scale is rounded to
//     fp16 once (bf16 results, which have 8 bits: it moves the error against 64 bits
//     from 0.0016 to 0.0017), or kept as a sum of two fp16 numbers, 22 bits (fp32 and
//     fp16 results, two products). These products are scaled by the largest value
//     scale that the row has seen: a key's share of a result is kept to 2^-34 of the
//     largest value that the row sees.
// Queries are scaled by a power of two to below 2^15; fp32 queries are the sum of
// two fp16 numbers, 22 bits.
//
// Few rows read every key once: bound by HBM and by the unpacking beside it. The
// cache goes to LDS by direct loads, a ring of steps for each wave, so that no
// register holds what is on its way, and waves share nothing until their sums are
// joined. 37 requests of up to 8192 keys, 32 heads over 8 of 128, bf16: 45.9 us, 179
// MB at 3.9 TB/s, with the vector units busy for 61 % of it; 32767 keys of 32 heads,
// fp32: 42.2 us, 3.6 TB/s, 73 % (two products for each of bf16's). (The last-level
// cache holds some of these caches from call to call.) One request of 1000 keys: 12.6
// us, a chain of launch, lengths, table, keys and sums in one workgroup a head.
// Prompts of a few hundred tokens run here too, where the kernel of
// attention_kv4_prompt.hip would leave most of the chip without a workgroup.
#include <algorithm>
#include <cmath>

#include "attention_common.h"

namespace pfng {
namespace {

constexpr int kRows = 16, kStep = 32;
constexpr int kMostParts = 256;  // of a row's keys

// A wave's keys come through a ring of LDS that only it reads and writes: stages of 32 tokens, as they lie in the cache.
template <int D>
struct Ring {
    static constexpr int NB = D / 32;
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr int kValues = 16 * D, kKeyScales = 32 * D, kValueScales = kKeyScales + 64 * NB;  // keys at 0
    static constexpr int kStage = kValueScales + 64 * NB;
    static constexpr int kHalf = 8 * D;                                // bytes of 16 tokens' keys
    static constexpr int kCopies = (D == 64 ? 2 : D / 32) + (D == 128 ? 2 : 1);  // instructions of a stage
};

// max over the four lane groups of a row
__device__ __forceinline__ float rows_max(float v) {
    v = fmaxf(v, xor_shfl<16>(v));
    return fmaxf(v, xor_shfl<32>(v));
}
__device__ __forceinline__ float rows_sum(float v) {
    v += xor_shfl<16>(v);
    return v + xor_shfl<32>(v);
}

// What one lane takes of a stage: for the scores, then for the values.
template <int D>
struct Keys {
    uint32_t k[2][D / 32];     // tile t: token 8(n / 4) + 4t + n % 4, slice g of every block
    f16x8 scale[D / 32];       // of tokens 8g..8g+7 [token][block]
};
template <int D>
struct Values {
    uint32_t v[D / 16];        // tokens 8g..8g+7, lane n's bytes
    f16x8 scale[D / 32];       // their scales [token][block]
    uint32_t top[D / 128 + 1]; // this lane's share of the stage's value scales, two or four to a lane
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t *dst, const uint8_t *src) {
    if constexpr (N == 2) {
        const uint2 t = *reinterpret_cast<const uint2 *>(src);
        dst[0] = t.x, dst[1] = t.y;
    } else {
        #pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 t = *reinterpret_cast<const uint4 *>(src + 16 * i);
            dst[4 * i] = t.x, dst[4 * i + 1] = t.y, dst[4 * i + 2] = t.z, dst[4 * i + 3] = t.w;
        }
    }
}

// Waves of a CU: what the registers of the sums leave.
constexpr int row_waves(int head_dim, bool fp32) {
    return head_dim == 256 ? 8 : head_dim == 128 || fp32 ? 12 : 16;
}

template <int D, class T, int kWaves>
__global__ __launch_bounds__(64 * kWaves, row_waves(D, sizeof(T) == 4) / kWaves) void attention_kv4_kernel(
    AttendArgs a) {
    constexpr int NB = D / 32, kTiles = D / 16;
    constexpr int kQ = std::is_same<T, float>::value ? 2 : 1;   // fp16 parts of a query
    constexpr int kP = std::is_same<T, __bf16>::value ? 1 : 2;  // of a probability
    constexpr int kPad = D + 4;
    using R = Ring<D>;
    extern __shared__ __align__(16) uint8_t lds[];  // the waves' rings; then their sums
    float (*lds_out)[kRows][kPad] = reinterpret_cast<float (*)[kRows][kPad]>(lds);
    __shared__ float lds_m[kWaves][kRows], lds_l[kWaves][kRows];
    static_assert(kWaves * kRows * kPad * 4 <= kWaves * R::kStages * R::kStage, "the sums fit where the rings were");

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t at = blockIdx.x;
    const int head = split_off(at, a.by_kv_heads), tile0 = split_off(at, a.by_tiles);
    const int request = split_off(at, a.by_requests), split = at;

    const int group = a.q_heads / a.kv_heads;
    const Request rq = request_of(a, request);
    if (rq.added < a.least || rq.added > a.most) return;
    const int32_t *table = a.table + request * a.table_stride;
    const int64_t page_bytes = kv_page_bytes(a.page_size, D), half_bytes = page_bytes * a.kv_heads;
    const uint8_t *cache = a.cache + head * page_bytes;
    const uint32_t rows = uint32_t(rq.added) * group;  // below 2^31

    for (uint32_t tile = tile0; tile * uint64_t(kRows) < rows; tile += a.tiles) {
        const uint32_t row = tile * kRows + n, row_end = min(rows, (tile + 1) * kRows);
        const bool row_on = row < rows;
        const int i_first = quotient(tile * kRows, a.by_group), i_last = quotient(row_end - 1, a.by_group);
        const int i_row = row_on ? quotient(row, a.by_group) : i_last;
        const int q_head = head * group + (row_on ? int(row) - i_row * group : 0);

        const int key_lo = row_first(a, rq, i_first) & ~(kStep - 1);
        const int key_hi = row_last(a, rq, i_last);
        const int steps = key_hi > key_lo ? (key_hi - key_lo + kStep - 1) / kStep : 0;
        // parts of the size that the longest request's have, so that no workgroup is left with little
        const int per = steps <= a.per * a.parts ? a.per : (steps + a.parts - 1) / a.parts;
        const int used = (steps + per - 1) / per;
        if (split >= max(used, 1)) continue;
        const int step0 = split * per, step1 = min(steps, step0 + per);
        const int last_n = row_last(a, rq, i_row), first_n = row_first(a, rq, i_row);
        // keys every row of the tile sees
        const int all_first = row_first(a, rq, i_last), all_last = row_last(a, rq, i_first);

        // The pages of a step's first and last 16 tokens; past the last step those of the last. A wave looks up those of
        // its next 64 steps at once, a lane each (one lookup a step would keep every step's LDS reads waiting for it:
        // their counter is that of scalar loads).
        struct Pages {
            int first, last;
        };
        int first_pages = 0, last_pages = 0;
        auto pages_of = [&](int i) __attribute__((always_inline)) -> Pages {  // of this wave's i-th step, in order
            if (i % 64 == 0) {
                const int key0 = key_lo + min(step0 + wave + (i + lane) * kWaves, steps - 1) * kStep, end = a.max_pages - 1;
                first_pages = table[min(key0 >> a.page_shift, end)];
                last_pages = table[min((key0 + 16) >> a.page_shift, end)];
                // waited for here, and not in each step
                asm volatile("" : "+v"(first_pages), "+v"(last_pages));
            }
            return {__builtin_amdgcn_readlane(first_pages, i % 64), __builtin_amdgcn_readlane(last_pages, i % 64)};
        };
        auto there = [&](int page) { return (uint32_t)page < (uint64_t)a.pages; };
        // Copies a step into its stage: R::kCopies instructions, each lane 4 or 16 bytes of a run within one page. Past
        // the last step it copies the last again, so that there are always as many.
        auto copy = [&](int step, Pages pages, uint8_t *stage) __attribute__((always_inline)) {
            const int key0 = key_lo + min(step, steps - 1) * kStep;
            const int tok0 = key0 & (a.page_size - 1), tok1 = (key0 + 16) & (a.page_size - 1);
            const uint8_t *p0 = cache + int64_t(there(pages.first) ? pages.first : 0) * 2 * half_bytes;
            const uint8_t *p1 = cache + int64_t(there(pages.last) ? pages.last : 0) * 2 * half_bytes;
            auto copy16 = [&](const uint8_t *from, int at) __attribute__((always_inline)) {
                __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void *)(stage + at), 16, 0, 0);
            };
            // nibbles: a token's D / 2 bytes, 16 tokens one after another, of keys and of values
            const uint8_t *n0 = p0 + tok0 * (D / 2), *n1 = p1 + tok1 * (D / 2);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int64_t away = half * half_bytes;
                if constexpr (D == 64) {
                    copy16((lane < 32 ? n0 : n1) + away + 16 * (lane & 31), half * R::kValues);
                } else {
#pragma unroll
                    for (int i = 0; i < R::kHalf / 1024; ++i) {
                        copy16(n0 + away + 1024 * i + 16 * lane, half * R::kValues + 1024 * i);
                        copy16(n1 + away + 1024 * i + 16 * lane, half * R::kValues + R::kHalf + 1024 * i);
                    }
                }
            }
            // scales: 32 NB bytes of 16 tokens
            const int plane = a.page_size * (D / 2);
            const uint8_t *s0 = p0 + plane + tok0 * NB * 2, *s1 = p1 + plane + tok1 * NB * 2;
            if constexpr (D == 128) {
                const uint8_t *from = (lane < 32 ? s0 : s1) + 4 * (lane & 31);
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    __builtin_amdgcn_global_load_lds(
                        from + half * half_bytes,
                        (__attribute__((address_space(3))) void *)(stage + (half ? R::kValueScales : R::kKeyScales)), 4, 0, 0);
            } else {
                constexpr int kEach = 2 * NB;  // bytes a lane: 16 lanes a run, both runs of keys, then of values
                const uint8_t *from = (lane & 16 ? s1 : s0) + (lane & 32 ? half_bytes : 0) + kEach * (lane & 15);
                auto *to = (__attribute__((address_space(3))) void *)(stage + R::kKeyScales);
                if constexpr (D == 64) __builtin_amdgcn_global_load_lds(from, to, 4, 0, 0);
                else __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
            }
        };
        auto take_keys = [&](const uint8_t *stage) __attribute__((always_inline)) -> Keys<D> {
            Keys<D> s;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                load_words<NB>(s.k[t], stage + (8 * (n >> 2) + 4 * t + (n & 3)) * (D / 2) + g * 4 * NB);
#pragma unroll
            for (int i = 0; i < NB; ++i)
                s.scale[i] = *reinterpret_cast<const f16x8 *>(stage + R::kKeyScales + 16 * NB * g + 16 * i);
            return s;
        };
        auto take_values = [&](const uint8_t *stage) __attribute__((always_inline)) -> Values<D> {
            Values<D> s;
#pragma unroll
            for (int i = 0; i < NB / 2; ++i)
                load_words<4>(&s.v[4 * i], stage + R::kValues + 4 * D * g + 16 * n + 256 * i);
            const uint8_t *scales = stage + R::kValueScales + 16 * NB * g;
#pragma unroll
            for (int i = 0; i < NB; ++i) s.scale[i] = *reinterpret_cast<const f16x8 *>(scales + 16 * i);
            // two scales a lane (four at D = 256; at D = 64 two lanes have the same ones)
#pragma unroll
            for (int i = 0; i < (NB + 3) / 4; ++i)
                s.top[i] = *reinterpret_cast<const uint32_t *>(scales + 4 * (n % (4 * NB)) + 64 * i);
            return s;
        };

        // the first steps, on their way while the queries are
        uint8_t *ring = lds + wave * (R::kStages * R::kStage);
        Pages pages[R::kStages] = {};
        if (step0 + wave < step1)
#pragma unroll
            for (int i = 0; i < R::kStages; ++i) {
                pages[i] = pages_of(i);
                copy(step0 + wave + i * kWaves, pages[i], ring + i * R::kStage);
            }

        const uint32_t magic = magic_bits();
        // the row's query, scaled by a power of two into fp16
        f16x8 q[kQ][NB];
        f32x4 start[NB];
        float to_log2;
        {
            f32x8 x[NB];
            float mag = 0.0f;
            const T *src = static_cast<const T *>(a.q) + int64_t(rq.begin + i_row) * a.q_stride + int64_t(q_head) * D;
            #pragma unroll
            for (int b = 0; b < NB; ++b) {
                x[b] = load8(src + 32 * b + 8 * g);
                #pragma unroll
                for (int e = 0; e < 8; ++e) mag = fmaxf(mag, fabsf(x[b][e]));
            }
            mag = rows_max(mag);
            const int exponent = mag > 0.0f && mag < INFINITY ? max(-100, ilogbf(mag)) : 0;
            const float factor = ldexpf(1.0f, 14 - exponent);
            // (past the largest number only with bf16 queries of 1e36 and more, whose scores any factor tells apart)
            to_log2 = ldexpf(a.scale_log2, exponent - 14 + (kP == 1 ? 24 : 0));
            to_log2 = fminf(fmaxf(to_log2, -0x1.fffffep127f), 0x1.fffffep127f);
            #pragma unroll
            for (int b = 0; b < NB; ++b) {
                float sum = 0.0f;
                #pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = x[b][e] * factor;
                    const _Float16 hi = (_Float16)v;
                    const _Float16 lo = (_Float16)(v - (float)hi);
                    // the nibbles of elements 2, 3, 6 and 7 stay four bits up
                    const _Float16 down = kP == 1 && (e & 2) ? (_Float16)0.0625f : (_Float16)1.0f;
                    q[0][b][e] = hi * down;
                    sum += (float)hi;
                    if constexpr (kQ == 2) {
                        q[1][b][e] = lo * down;
                        sum += (float)lo;
                    }
                }
                const float c = rows_sum(sum) * (-8.0f * 0x1p-24f);
                start[b] = f32x4{c, c, c, c};
            }
        }

        f32x4 o[kTiles] = {};
        // Probabilities are 2^(score - base) with a whole number for base, so that moving it is exact. It moves when a
        // score is 3 above it, and at the row's first: a row's largest scores come early, and moving costs as many
        // products as the row has elements. (Past 2^24 the base itself is rounded, to what fp32 tells apart of the
        // scores; what it moves by is not, so that the row's largest probability is 1 all the same.)
        float base = 0.0f, l = 0.0f, limit = -INFINITY;
        // Exponent field of the largest value scale that the row has seen: the products of its probabilities (up to 8) and
        // scales are scaled by 2^(25 - top), to below 2^14. Each row has its own: by a token that it does not see, its
        // products could fall below what fp16 holds.
        int top = 1, least_top = 1;  // least_top: of the tile's rows
        float up = 0x1p24f;

        auto multiply = [&](int step, Pages pages, const uint8_t *stage, auto refill) __attribute__((always_inline)) {
            const int key0 = key_lo + step * kStep;
            const bool page_ok = g < 2 ? there(pages.first) : there(pages.last);
            const bool whole =
                key0 >= all_first && key0 + kStep <= all_last && there(pages.first) && there(pages.last);
            const Keys<D> keys = take_keys(stage);

            // exponents of tokens 8g + 4t + i. A SIMD serves the waves that are here before those at their values: 2 % over 42
            // sizes (37 requests of 1000 keys, 32 heads over 8 of 128, bf16 20.8 -> 20.0 us; the other way round is no
            // faster than without).
            __builtin_amdgcn_s_setprio(1);
            float x[8];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 s = {};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const f16x8 kf = kP == 1 ? key_subnormals(keys.k[t][b]) : key_numbers(keys.k[t][b], magic);
                    const f32x4 first = kP == 1 ? start[b] : f32x4{};
                    f32x4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[0][b], first, 0, 0, 0);
                    if constexpr (kQ == 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[1][b], acc, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = (4 * t + i) * NB + b;
                        s[i] = __builtin_fmaf(acc[i], (float)keys.scale[at / 8][at % 8], s[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * t + i] = __builtin_fmaf(s[i], to_log2, -base);
            }
            Values<D> values = take_values(stage);
            refill();
            if (!whole) {
                // hidden tokens: no probability, and a scale of 0, for theirs may be anything
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = key0 + 8 * g + i;
                    if (!(page_ok && key >= first_n && key < last_n)) {
                        x[i] = -INFINITY;
#pragma unroll
                        for (int b = 0; b < NB; ++b) values.scale[(i * NB + b) / 8][(i * NB + b) % 8] = (_Float16)0.0f;
                    }
                }
            }

            float mx = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) mx = __builtin_elementwise_maximum(mx, x[i]);
            if (__any(mx > limit)) {
                mx = __builtin_elementwise_maximum(mx, xor_shfl<16>(mx));
                mx = __builtin_elementwise_maximum(mx, xor_shfl<32>(mx));
                const bool first = limit == -INFINITY;
                const float by = mx > (first ? -INFINITY : 0.0f) ? rintf(mx) : 0.0f;
                if (mx > -INFINITY) limit = 3.0f;
                const float alpha = first ? 1.0f : exp2_of(-by);
                base += by;
                l *= alpha;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) o[t] *= alpha;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] -= by;
            }
            // whether a value scale of the step may be larger than a row has seen
            int largest = 0;
#pragma unroll
            for (int i = 0; i < (NB + 3) / 4; ++i) {
                const uint32_t two = values.top[i] & 0x7fff7fffu;
                largest = max(largest, int(max(two & 0xffffu, two >> 16)));
            }
            if (__any(largest >= (least_top + 1) << 10)) {
                // of what this row sees (hidden tokens' scales are 0 here); one that is not finite becomes negative and
                // does not count
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                s16x8 most = {};
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    most = __builtin_elementwise_max(most, (__builtin_bit_cast(s16x8, values.scale[i]) & (short)0x7fff) + (short)0x0400);
                int seen = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) seen = max(seen, (int)most[i]);
                seen = max(top, (seen >> 10) - 1);
                seen = max(seen, xor_shfl<16>(seen));
                seen = max(seen, xor_shfl<32>(seen));
                const float down = ldexpf(1.0f, top - seen);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) o[t] *= down;
                top = seen;
                up = ldexpf(1.0f, 25 - top);
                least_top = butterfly<8>(top, [](int x, int y) { return min(x, y); });
            }

            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = exp2_of(x[i]);
                l += p[i];
                p[i] *= up;
            }
            // O^T += V^T (P d)^T, block by block
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f16x8 ph, pl;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = (float)values.scale[(i * NB + b) / 8][(i * NB + b) % 8];
                    ph[i] = (_Float16)__builtin_fmaf(p[i], d, 0.0f);
                    if constexpr (kP == 2) pl[i] = (_Float16)__builtin_fmaf(p[i], d, -(float)ph[i]);
                }
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // bytes b of tokens 2i and 2i + 1
                    const int at0 = 2 * i * NB + b, at1 = at0 + NB;
                    const uint32_t pair = __builtin_amdgcn_perm(values.v[at1 / 4], values.v[at0 / 4],
                                                                0x0c000c00u | ((4u + at1 % 4) << 16) | (at0 % 4));
                    lo[i] = low_numbers(pair, magic);
                    hi[i] = high_numbers(pair, magic);
                }
                const f16x8 v0 = as_f16x8(lo[0], lo[1], lo[2], lo[3]), v1 = as_f16x8(hi[0], hi[1], hi[2], hi[3]);
                o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph, o[2 * b], 0, 0, 0);
                o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph, o[2 * b + 1], 0, 0, 0);
                if constexpr (kP == 2) {
                    o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl, o[2 * b], 0, 0, 0);
                    o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl, o[2 * b + 1], 0, 0, 0);
                }
            }
        };

        // kStages - 1 steps are on their way while one is multiplied: copies complete in order, so that at most the
        // later stages' may be outstanding when a stage is read.
        if (step0 + wave < step1) {
            int stage = 0, ahead = R::kStages;
            for (int step = step0 + wave; step < step1; step += kWaves) {
                const Pages next = pages_of(ahead++);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R::kStages - 1) * R::kCopies) : "memory");
                multiply(step, pages[0], ring + stage, [&]() __attribute__((always_inline)) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the stage may be filled again
                    copy(step + R::kStages * kWaves, next, ring + stage);
                });
#pragma unroll
                for (int i = 0; i + 1 < R::kStages; ++i) pages[i] = pages[i + 1];
                pages[R::kStages - 1] = next;
                stage = stage + R::kStage == R::kStages * R::kStage ? 0 : stage + R::kStage;
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy lands where the sums will be
        }
        __syncthreads();

        // join the waves
        const float whole_l = rows_sum(l), back = ldexpf(1.0f, top - 25);
        #pragma unroll
        for (int t = 0; t < kTiles; ++t) *reinterpret_cast<f32x4 *>(&lds_out[wave][n][16 * t + 4 * g]) = o[t] * back;
        if (g == 0) {
            lds_m[wave][n] = limit == -INFINITY ? -INFINITY : base;
            lds_l[wave][n] = whole_l;
        }
        __syncthreads();
        constexpr int kRowLanes = 4 * kWaves;  // threads that join a row
        const int r = tid / kRowLanes, part = tid % kRowLanes;
        const uint32_t out_row = tile * kRows + r;
        if (out_row < rows) {
            float big = lds_m[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) big = fmaxf(big, lds_m[w][r]);
            const float to = big == -INFINITY ? 0.0f : big;
            float weight[kWaves], sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                weight[w] = exp2_of(lds_m[w][r] - to);
                sum += weight[w] * lds_l[w][r];
            }
            const int out_i = quotient(out_row, a.by_group);
            const int token = rq.begin + out_i, oh = head * group + int(out_row) - out_i * group;
            const int64_t out_at = int64_t(token) * a.q_heads + oh;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            for (int d = 4 * part; d < D; d += 4 * kRowLanes) {
                f32x4 v = {};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) v += weight[w] * *reinterpret_cast<const f32x4 *>(&lds_out[w][r][d]);
                if (used > 1) {
                    *reinterpret_cast<f32x4 *>(a.part_out + (out_at * a.splits + split) * D + d) = v;
                } else {
                    if (sum == 0.0f) v = f32x4{};
                    store4(static_cast<T *>(a.out) + token * a.out_stride + int64_t(oh) * D + d, v * inv);
                }
            }
            if (part == 0 && a.splits > 1) {
                if (used > 1) {
                    a.part_ml[(out_at * a.splits + split) * 2] = big;
                    a.part_ml[(out_at * a.splits + split) * 2 + 1] = sum;
                }
                if (split == 0) a.part_count[out_at] = used;
            }
        }
        __syncthreads();
    }
}

// Joins the parts of one (token, head): 16 lanes, four elements each and 64 on.
template <int D, class T>
__global__ __launch_bounds__(256) void attention_kv4_join_kernel(AttendArgs a) {
    const int64_t row = int64_t(blockIdx.x) * 16 + threadIdx.x / 16;
    if (row >= a.tokens * a.q_heads) return;
    const int count = min(a.part_count[row], a.splits);
    if (count <= 1) return;
    const float *ml = a.part_ml + row * a.splits * 2;
    float big = -INFINITY, sum = 0.0f;
    for (int s = 0; s < count; ++s) big = fmaxf(big, ml[2 * s]);
    const float base = big == -INFINITY ? 0.0f : big;
    f32x4 v[D / 64] = {};
    for (int s = 0; s < count; ++s) {
        const float w = exp2_of(ml[2 * s] - base);
        sum += w * ml[2 * s + 1];
        #pragma unroll
        for (int i = 0; i < D / 64; ++i)
            v[i] += w * *reinterpret_cast<const f32x4 *>(a.part_out + (row * a.splits + s) * D + 64 * i +
                                                         4 * (threadIdx.x % 16));
    }
    const int64_t token = row / a.q_heads;
    T *dst = static_cast<T *>(a.out) + token * a.out_stride + (row - token * a.q_heads) * D + 4 * (threadIdx.x % 16);
    #pragma unroll
    for (int i = 0; i < D / 64; ++i) store4(dst + 64 * i, sum == 0.0f ? f32x4{} : v[i] / sum);
}

// The same with a workgroup a row, for many parts: a thread a part for the weights, then D / 4 lanes by kGroups parts.
template <int D, class T>
__global__ __launch_bounds__(256) void attention_kv4_join_many_kernel(AttendArgs a) {
    constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
    __shared__ float weight[kMostParts], wave_max[4], wave_sum[4];
    __shared__ f32x4 sums[kGroups][kLanes];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, count = min(a.part_count[row], a.splits);
    if (count <= 1) return;
    const float *ml = a.part_ml + row * a.splits * 2;
    const float m = tid < count ? ml[2 * tid] : -INFINITY, l = tid < count ? ml[2 * tid + 1] : 0.0f;
    const float most = butterfly<32>(m, [](float x, float y) { return fmaxf(x, y); });
    if (tid % 64 == 0) wave_max[tid / 64] = most;
    __syncthreads();
    const float big = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
    const float w = exp2_of(m - (big == -INFINITY ? 0.0f : big));
    weight[tid] = w;
    const float part_sum = butterfly<32>(w * l, [](float x, float y) { return x + y; });
    if (tid % 64 == 0) wave_sum[tid / 64] = part_sum;
    __syncthreads();
    const float sum = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    const int e = tid % kLanes, group = tid / kLanes;
    f32x4 v = {};
    for (int s = group; s < count; s += kGroups)
        v += weight[s] * *reinterpret_cast<const f32x4 *>(a.part_out + (row * a.splits + s) * D + 4 * e);
    sums[group][e] = v;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) v += sums[i][e];
    const int64_t token = row / a.q_heads;
    store4(static_cast<T *>(a.out) + token * a.out_stride + (row - token * a.q_heads) * D + 4 * e,
           sum == 0.0f ? f32x4{} : v / sum);
}

template <int D, class T, int W>
hipError_t launch_waves(const AttendArgs &a, hipStream_t s) {
    const int64_t grid = int64_t(a.requests) * a.tiles * a.parts * a.kv_heads;
    attention_kv4_kernel<D, T, W><<<dim3((unsigned)grid), 64 * W, W * Ring<D>::kStages * Ring<D>::kStage, s>>>(a);
    return hipGetLastError();
}

template <int D, class T>
hipError_t launch_typed(const AttendArgs &args, const AttendPlan &plan, int type, hipStream_t s) {
    AttendArgs a = args;
    for (int i = 0; i < plan.launches; ++i) {
        const AttendLaunch &l = plan.launch[i];
        a.tiles = l.tiles, a.parts = l.parts, a.per = l.per, a.least = l.least, a.most = l.most;
        a.by_tiles = Divisor(l.tiles);
        const hipError_t e = l.prompt       ? launch_attention_kv4_prompt(a, type, D, s)
                             : l.waves == 8 ? launch_waves<D, T, 8>(a, s)
                                            : launch_waves<D, T, 4>(a, s);
        if (e != hipSuccess) return e;
    }
    if (a.splits == 1) return hipSuccess;
    const int64_t rows = a.tokens * a.q_heads;
    // By 16 lanes and by a workgroup a row, heads of 128: 1024 rows of 4 parts 4.0 and 3.9 us, of 8 5.5 and 3.9, of 16 8.8
    // and 3.9; 4096 rows 4.6 and 5.6, 7.1 and 5.8, 9.8 and 7.2; 16384 rows 7.3 and 16.6, 13.8 and 17.0, 19.0 and 21.3.
    if (a.splits > 4 && rows <= 512 * a.splits) attention_kv4_join_many_kernel<D, T><<<dim3((unsigned)rows), 256, 0, s>>>(a);
    else attention_kv4_join_kernel<D, T><<<dim3((unsigned)((rows + 15) / 16)), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const AttendArgs &a, const AttendPlan &plan, int type, hipStream_t s) {
    switch (type) {
    case 0: return launch_typed<D, float>(a, plan, type, s);
    case 1: return launch_typed<D, __bf16>(a, plan, type, s);
    default: return launch_typed<D, _Float16>(a, plan, type, s);
    }
}

// The kernel, the parts of the keys and the waves of a workgroup are chosen by models of the kernels' measured times, in ns
// (one MI355X; fitted to both kernels at 840 sizes in 1 to 48 parts: requests 1 to 32 of equal lengths, new tokens 1 to
// 4096, up to 16384 keys, heads of 64, 128 and 256, fp32 and bf16). With the kernels as they are, what they choose takes
// 2.5 % longer than the fastest of both kernels, both numbers of waves and 11 of parts (geometric mean over 603 sizes of
// fp32, bf16 and fp16; 46 % at worst: 16 fp32 tokens of 1016 keys at heads of 256, 22.5 us in one launch, 15.4 in 8 parts).
struct Sizes {
    int type, q_heads, kv_heads, head_dim, cus;
    int64_t requests, max_added, max_length;  // of the requests that the launch is for
    int64_t launched;                         // all requests times key heads: each has workgroups, if only to find no rows
    int64_t joined;                           // rows of all: parts are joined by 16 threads each
    bool causal;
};
struct Planned {
    AttendLaunch plan;
    double ns = INFINITY;
};
constexpr int kFew = 4;                              // new tokens of a running request
constexpr int64_t kMixedBytes = int64_t(256) << 20;  // of parts, which have places for every row, for those of a few
constexpr int kParts[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128, 192, kMostParts};

// Row tiles of `rows` rows, keys in steps of `keys`.
struct Shape {
    int tiles;             // of the longest request, as launched
    int64_t steps;         // of its last row tile
    double groups, average;  // row tiles and heads of all, steps of one on average
};
Shape shape_of(const Sizes &z, int64_t tile_rows, int64_t keys) {
    const int64_t rows = z.max_added * (z.q_heads / z.kv_heads), heads = std::max<int64_t>(1, z.requests * z.kv_heads);
    const int64_t tiles = std::max<int64_t>(1, (rows + tile_rows - 1) / tile_rows);
    Shape s;
    // a workgroup takes every tiles-th tile: fewer where the grid would pass 2^22 workgroups
    s.tiles = (int)std::min<int64_t>(tiles, std::max<int64_t>(1, (int64_t(1) << 22) / std::max<int64_t>(1, z.launched)));
    s.steps = std::max<int64_t>(1, (z.max_length + keys - 1) / keys);
    s.groups = (double)heads * tiles;
    // of the first and the last row tile, half and half
    const int64_t hidden =
        std::max<int64_t>(0, std::min(z.max_added, z.max_length) - tile_rows * z.kv_heads / z.q_heads) / 2;
    s.average = (double)std::max<int64_t>(1, ((z.causal ? z.max_length - hidden : z.max_length) + keys - 1) / keys);
    return s;
}

// HIP takes fewer than 2^32 threads in a launch. (One part of 4 waves always fits: launched is below 2^24.)
bool fits(const Sizes &z, const Shape &s, int64_t parts, int threads) {
    return z.launched * s.tiles * parts * threads < int64_t(1) << 32 && (parts == 1 || z.joined < int64_t(1) << 27);
}

// The parts that a row tile has on average, where the longest has n of `per` steps.
double parts_of(double average, int64_t n, int64_t per) { return n == 1 ? 1 : std::min<double>(n, average / per + 0.5); }

// Workgroups in `rounds` rounds, of `each` ns on average: the last round is as long as its workgroups are alike, by `tail`.
double rounds_time(const Shape &s, int64_t n, double rounds, double each, double tail) {
    const double even = n > 1 ? 1 : std::max(0.0, 2 * s.average / s.steps - 1);
    return each * (rounds + (std::ceil(rounds) - rounds) * even * tail);
}

// attention_kv4_prompt.hip: a workgroup has a CU to itself, starts, reads its first tile and ends in 8.6 us (6 where another
// one follows), and takes 1.7 us a tile (with the keys, values and probabilities of fp32 and fp16 in two parts 3.4 at heads
// of 64, 3.8 at 128, 3 at 256). Parts are written and read in fp32 at 4 TB/s and joined by a launch of 2.5 us.
Planned plan_prompt(const Sizes &z) {
    const int64_t tile_rows = prompt_tile_rows(z.head_dim), rows = z.max_added * (z.q_heads / z.kv_heads);
    const Shape s = shape_of(z, tile_rows, prompt_tile_keys(z.head_dim));
    const double step = z.type == 1 ? 1720 : z.head_dim == 64 ? 3350 : z.head_dim == 128 ? 3750 : 2950, start = 8600;
    Planned best;
    for (const int64_t n : kParts) {
        if (n > s.steps || !fits(z, s, n, 2 * (int)tile_rows)) break;
        const int64_t per = (s.steps + n - 1) / n;
        const double parts = parts_of(s.average, n, per), rounds = s.groups * parts / z.cus;
        double ns = start + per * step;
        if (rounds > 1) ns = std::max(ns, rounds_time(s, n, rounds, 0.7 * start + s.average / parts * step, 1.0));
        if (n > 1) ns += 2500 + s.groups * parts * std::min<int64_t>(rows, tile_rows) * z.head_dim * 8 / 4000;
        if (ns < best.ns) {
            best.ns = ns;
            best.plan.prompt = true, best.plan.tiles = s.tiles;
            best.plan.parts = (int)((s.steps + per - 1) / per), best.plan.per = (int)per;
        }
        if (rounds > 8) break;
    }
    return best;
}

// This file's kernel: a workgroup of 4 or 8 waves starts and ends in 3.5 us and 15 ns for each element of a head, a call in
// 2 us more. A wave takes 0.7 us and 4.5 ns an element for a step (1.4 times that with two parts to a number) where the CU
// is not full, and the CU 1.4 ns an element (1.9) for each wave's step. Joining parts takes 4 us and their traffic, and
// 2 us more of a host that a call in one launch keeps waiting (1000 keys, 32 heads over 8 of 128: 12.8 us in one part, 7.3
// + 3.7 in eight; 14.5 and 18.6 called from Python). 8 waves are for those that all find a CU. Requests are of any length
// up to the longest, which is all that is known: a third of the weight has all alike, the rest half of it on average (37
// requests of up to 8192 keys, 32 heads over 8 of 128: 66, 59, 55, 46, 52 and 51 us in 1, 2, 3, 4, 5 and 8 parts).
Planned plan_rows(const Sizes &z) {
    const Shape s = shape_of(z, kRows, kStep);
    const bool two = z.type != 1;
    const double alone = (700 + 4.5 * z.head_dim) * (two ? 1.4 : 1.0), busy = z.head_dim * (two ? 1.9 : 1.4);
    const double start = 3500 + 15 * z.head_dim;
    const double row_bytes = double(z.requests) * z.max_added * z.q_heads * z.head_dim * 8;
    double least = INFINITY;
    Planned best;
    for (const int64_t n : kParts) {
        if (n > 1 && (s.steps < 4 * n || !fits(z, s, n, 256))) break;
        const int64_t per = (s.steps + n - 1) / n;
        for (const int waves : {4, 8}) {
            const int beside = std::max(1, row_waves(z.head_dim, z.type == 0) / waves);  // workgroups of a CU
            if (waves == 8 && (s.groups * n > z.cus * beside || !fits(z, s, n, 512))) break;
            auto time = [&](double average) {
                const double parts = parts_of(average, n, per), rounds = s.groups * parts / z.cus / beside;
                const double shared = std::min<double>(beside, std::max(1.0, rounds * beside));
                double ns = start + (per + waves - 1) / waves * std::max(alone, shared * waves * busy);
                if (rounds > 1) {
                    const double each = std::ceil(average / parts / waves) * std::max(alone, beside * waves * busy);
                    ns = std::max(ns, rounds_time(s, n, rounds, start + each, 0.5));
                }
                return ns + 2000 + (n > 1 ? 6000 + row_bytes * parts / 4000 : 0);
            };
            const double alike = time(s.average);
            const double ns = z.requests > 1 ? (alike + 2 * time(std::max(1.0, s.average / 2))) / 3 : alike;
            if (ns < least) {
                least = ns, best.ns = alike;
                best.plan.tiles = s.tiles, best.plan.waves = waves;
                best.plan.parts = (int)((s.steps + per - 1) / per), best.plan.per = (int)per;
            }
        }
        if (s.groups * n > 32 * z.cus) break;
    }
    return best;
}

}  // namespace

AttendPlan plan_attention(int type, int64_t tokens, int64_t requests, int q_heads, int kv_heads, int head_dim,
                          int64_t max_added, int64_t max_length, bool causal, int cus) {
    Sizes z{type, q_heads, kv_heads, head_dim, cus, requests, max_added, max_length, requests * kv_heads, tokens * q_heads, causal};
    AttendPlan p;
    AttendLaunch &main = p.launch[0];
    // A step that serves new prompts and running requests has half of what max_added says, or less: a launch for each, or
    // running requests' long contexts would go through the prompts' tiles for a row or two (a prompt of 2048 beside 31
    // requests of 8192 keys, 32 heads over 8 of 128, bf16: 404 us in one, 136 in two; 512 beside 63 of 1024: 85, 47).
    const bool mixed = requests > 1 && max_added > kFew && tokens <= requests * max_added / 2;
    Sizes few = z;
    if (mixed) {
        few.max_added = 1;
        z.requests = std::max<int64_t>(1, std::min(requests, (tokens + max_added - 1) / max_added));
    }
    const Planned rows = plan_rows(z);
    main = rows.plan;
    if (max_added * (q_heads / kv_heads) > kRows) {
        const Planned prompt = plan_prompt(z);
        if (prompt.ns < rows.ns) main = prompt.plan;
    }
    p.splits = main.parts;
    if (mixed) {
        AttendLaunch &single = p.launch[p.launches++];
        single = plan_rows(few).plan;
        const int64_t part_bytes = std::max<int64_t>(1, tokens * q_heads * head_dim * 4);
        const int most = (int)std::max<int64_t>({1, main.parts, kMixedBytes / part_bytes});
        if (single.parts > most) {
            const int64_t steps = int64_t(single.parts) * single.per;
            single.parts = most, single.per = (int)((steps + most - 1) / most);
        }
        single.most = kFew, main.least = kFew + 1;
        p.splits = std::max(p.splits, single.parts);
    }
    return p;
}

hipError_t launch_attention_kv4(const AttendArgs &a, const AttendPlan &plan, int type, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 64: return launch_dim<64>(a, plan, type, s);
    case 128: return launch_dim<128>(a, plan, type, s);
    default: return launch_dim<256>(a, plan, type, s);
    }
}

}  // namespace pfng
