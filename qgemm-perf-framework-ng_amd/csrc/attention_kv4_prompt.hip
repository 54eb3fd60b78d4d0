// Attention of many new tokens over the paged 4-bit cache: the mathematics of
// attention_kv4.hip, shaped for matrix-instruction throughput.
//
// A workgroup takes 32 rows (query, head) of one key head for each of its waves
// and goes through the keys in tiles of KT. Its waves decode a tile together,
// half of them the keys, half the values, into LDS as fp16, in the order in which
// v_mfma_f32_16x16x32_f16 takes it (each operand is one 16-byte read a lane, the
// lanes one after another: no bank is asked twice); every wave then multiplies
// its rows with the whole tile, each operand twice, for rows 0..15 and 16..31.
// While one buffer is multiplied, the next tile is decoded into the other and the
// one after that is on its way from memory: one barrier a tile.
//
// S^T = K Q^T leaves lane (g = lane / 16, n = lane % 16) row n's scores of tokens
// 16t + 4g + 0..3 of tile t. Two tiles make the operand of O^T += V^T P^T, whose
// 32 values are placed in that order: the probabilities stay in their lane.
//
// 4096 tokens, 32 heads over 8 of 128, bf16: 152 to 157 us (more on cards that clock
// lower), 880 TFLOP/s; 1024 tokens after 15360 280 us, 950 TFLOP/s, where a large bf16
// product reaches 1212. In the first, the matrix units are busy for 37 % of the cycles,
// the vector units (exponentials, rounding, unpacking) for 51 %, LDS reads for 27 %; these
// add up more than they overlap. Decoding tiles beforehand, 64 rows a wave, tiles of
// twice the keys and other orders of the steps were measured and are no faster.
// Heads of 64 have half the products for each exponential: 5 prompts of 480 tokens
// after 1520, 24 heads, 51 us.
//
// Under load this card's clock goes by what it draws: on random numbers the
// 16x16x32 instruction sustains 2.0 PFLOP/s and 32x32x16 1.68 (its accumulators
// are read and written twice as often).
//
// For bf16 results, which have 8 bits, the operands have fp16's 11: the decoded keys and
// values (q - 8) * d (products with d below 2^-14 are exact: multiples of 2^-24 below
// 2^-10), the queries times scale and log2(e), and the probabilities, each rounded once.
// A score is off by up to 2^-11 of scale * sum |q k| by that, and the error against 64
// bits at prompts of 480 is 0.00174, where rounding the result alone makes 0.00166.
// fp32 and fp16 results take keys and values exactly, as a sum of two fp16 numbers, and
// the probabilities and fp32 queries to 22 bits in the same way: three products in the
// place of one (two for the scores of fp16, whose queries have no second part). Scores are summed from -base in fp32, so rounded at the size of base,
// for bf16 results; for the others base is taken off behind the sum. Sums of
// probabilities are in fp32 and, for bf16 results, of the rounded ones.
//
// Scales of 2^13 and more (values past 65504) would overflow: a token with one is
// decoded divided by 8, and alone (small scales would lose bits, and rows that do
// not see that token must not lose theirs). Its scores are multiplied by 8 within
// the exponent's product, its probabilities by 3 more in the exponent. Values whose
// scale is not finite are decoded as 0, and the rows that see them are set to NaN at
// the end. These, and pages outside the cache, mark the tile: only marked tiles look
// for them.
#include "attention_common.h"

namespace pfng {
namespace {

template <int D, class T, int W, int KT>
struct PromptShape {
    static constexpr int NB = D / 32;
    static constexpr bool kExact = !std::is_same<T, __bf16>::value;
    static constexpr int kParts = kExact ? 2 : 1;                     // fp16 parts of keys, values, probabilities
    static constexpr int kQ = std::is_same<T, float>::value ? 2 : 1;  // of queries
    // half of the threads decode the keys, the others the values: 16 bytes each (of values: a chunk), or twice that
    static constexpr int kChunkTokens = kv_chunk_tokens(D);
    static constexpr int kRowPieces = D / 32;                         // 16-byte pieces of a key row
    static constexpr int kPart = KT * D * 2;                          // LDS bytes of one part
    static constexpr int kBuffer = 2 * kParts * kPart;                // keys, then values
    static constexpr int kPieces = KT * kRowPieces / (32 * W);        // of 16 bytes, a thread's
    static constexpr int kRowLanes = 64 / kRowPieces;                 // tokens of 64 key pieces
    static_assert(kPieces >= 1 && kPieces * 32 * W == KT * kRowPieces && KT * D / 512 * 16 == KT * kRowPieces,
                  "whole pieces");
};

// What a thread keeps of the tile on its way: 16 bytes of nibbles and their scales.
struct Incoming {
    uint32_t w[4], scale[8];  // keys use one or two words of scales
    uint32_t check;           // of values: one of the scale words; the lanes of a chunk have them all between them
    bool page_ok;
};

// Exponent field of either half of a word of two scales at 28 or above: |d| >= 2^13 or not finite.
__device__ __forceinline__ bool large_scale(uint32_t two) {
    return ((two & (two << 1) & (two << 2)) & 0x40004000u) != 0;
}
__device__ __forceinline__ int exponent_of(uint32_t half) { return (half >> 10) & 31; }

// LDS reads are issued this many operands before the product that takes them (a read takes about as long as four
// products), each behind a product and pinned there: the compiler's own order, one read and a wait before each
// product, leaves the matrix units idle for most of the time.
constexpr int kAhead = 4;
__device__ __forceinline__ void pin_order() { __builtin_amdgcn_sched_barrier(0); }

template <int D, class T, int W, int KT>
__global__ __launch_bounds__(64 * W, 1) void attention_kv4_prompt_kernel(AttendArgs a) {
    using S = PromptShape<D, T, W, KT>;
    constexpr int NB = S::NB, kSub = KT / 16, kDepth = D / 16, kRows = 32 * W;
    // tiles of 16 keys that a wave has scores of at a time: as many as its registers hold
    constexpr int kPass = S::kExact || D == 256 ? 2 : 4;
    extern __shared__ __align__(16) uint8_t lds[];  // two buffers
    __shared__ int marked[2];                       // the step that last marked each buffer
    // of each token: what multiple of a score is added to it (0, or 7 of a divided one), and what to the exponents of the
    // probabilities
    __shared__ __align__(16) float score_more[2][KT], value_shift[2][KT];

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t at = blockIdx.x;
    // The longest rows first, and all parts that every row tile has before those that only the longest have: of 8
    // workgroups in a row each XCD gets one, so that each gets as many that find work. Requests take turns from tile to
    // tile: with fixed places, the row tiles of one long request among 16 all went to a quarter of each XCD (639 us, 200
    // this way); all tiles of a request in a row would end with the long tiles of the last one (8 x 1024 tokens 114 ->
    // 136 us).
    const int head = split_off(at, a.by_kv_heads);
    uint32_t turn = split_off(at, a.by_requests);
    const int tile0 = a.tiles - 1 - split_off(at, a.by_tiles), split = at;
    turn += tile0;
    const int request = split_off(turn, a.by_requests);

    const int group = a.q_heads / a.kv_heads;
    const Request rq = request_of(a, request);
    if (rq.added < a.least || rq.added > a.most) return;
    const int32_t *table = a.table + request * a.table_stride;
    const int64_t page_bytes = kv_page_bytes(a.page_size, D), half_bytes = page_bytes * a.kv_heads;
    const uint8_t *cache = a.cache + head * page_bytes;
    const uint32_t rows = uint32_t(rq.added) * group;  // below 2^31
    if (tid < 2) marked[tid] = -1;
    __syncthreads();

    for (uint32_t tile = tile0; tile * uint64_t(kRows) < rows; tile += a.tiles) {
        const uint32_t row_end = min(rows, (tile + 1) * kRows);
        const int i_first = quotient(tile * kRows, a.by_group), i_last = quotient(row_end - 1, a.by_group);
        const int key_lo = row_first(a, rq, i_first) & ~(KT - 1), key_hi = row_last(a, rq, i_last);
        const int steps = key_hi > key_lo ? (key_hi - key_lo + KT - 1) / KT : 0;
        // parts of the size that the longest request's have, so that no workgroup is left with little
        const int per = steps <= a.per * a.parts ? a.per : (steps + a.parts - 1) / a.parts;
        const int used = (steps + per - 1) / per;
        if (split >= max(used, 1)) continue;
        const int step0 = split * per, step1 = min(steps, step0 + per);

        // ---- from memory -----------------------------------------------------
        const bool keys = wave < W / 2;
        const int decoder = keys ? wave : wave - W / 2;
        // neighbouring lanes take neighbouring tokens of the keys, so that their 16-byte writes to LDS meet no bank
        // twice, and neighbouring lanes c of a chunk of values
        const int piece = lane / S::kRowLanes, c = lane % 16;
        auto token_of = [&](int u) -> int {
            return keys ? (decoder * S::kPieces + u) * S::kRowLanes + lane % S::kRowLanes
                        : ((decoder * S::kPieces + u) * 4 + lane / 16) * S::kChunkTokens;
        };
        struct Pages {
            int at[S::kPieces];
        };
        auto pages_of = [&](int step) -> Pages {
            Pages p;
#pragma unroll
            for (int u = 0; u < S::kPieces; ++u) {
                const int key = key_lo + min(step, steps - 1) * KT + token_of(u);
                p.at[u] = table[min(key >> a.page_shift, a.max_pages - 1)];
            }
            return p;
        };
        struct Tile {
            Incoming piece[S::kPieces];
        };
        auto load = [&](int step, Pages pages) __attribute__((always_inline)) -> Tile {
            Tile tile;
#pragma unroll
            for (int u = 0; u < S::kPieces; ++u) {
                Incoming &in = tile.piece[u];
                const int key = key_lo + min(step, steps - 1) * KT + token_of(u), token = key & (a.page_size - 1);
                in.page_ok = (uint32_t)pages.at[u] < (uint64_t)a.pages;
                const uint8_t *p =
                    cache + int64_t(in.page_ok ? pages.at[u] : 0) * 2 * half_bytes + (keys ? 0 : half_bytes);
                const uint4 w = *reinterpret_cast<const uint4 *>(
                    p + (keys ? kv_key_word(token, 0, 0, D) + 16 * piece : kv_value_bytes(token, c, D)));
                in.w[0] = w.x, in.w[1] = w.y, in.w[2] = w.z, in.w[3] = w.w;
                const uint8_t *s = p + kv_scale(a.page_size, token, 0, D);
                if (keys) {
                    // the words' blocks: all of the row's, at D = 256 the piece's half of them
                    if constexpr (NB == 2) {
                        in.scale[0] = *reinterpret_cast<const uint32_t *>(s);
                    } else {
                        const uint2 t = *reinterpret_cast<const uint2 *>(s + (NB == 8 ? 8 * (piece & 1) : 0));
                        in.scale[0] = t.x, in.scale[1] = t.y;
                    }
                } else {
                    const uint4 t = reinterpret_cast<const uint4 *>(s)[0], u4 = reinterpret_cast<const uint4 *>(s)[1];
                    in.scale[0] = t.x, in.scale[1] = t.y, in.scale[2] = t.z, in.scale[3] = t.w;
                    in.scale[4] = u4.x, in.scale[5] = u4.y, in.scale[6] = u4.z, in.scale[7] = u4.w;
                    in.check = reinterpret_cast<const uint32_t *>(s)[c & 7];
                }
            }
            return tile;
        };

        // the first tiles, on their way while the queries are
        Pages page = {};
        Tile in = {};
        if (step0 < step1) {
            page = pages_of(step0);
            in = load(step0, page);
            page = pages_of(step0 + 1);
        }

        // this wave's rows, this lane's two: n and 16 + n
        const uint32_t wave_row = tile * kRows + wave * 32;
        const bool wave_on = wave_row < rows;
        const uint32_t wave_end = min(rows, wave_row + 32);
        const int wave_i0 = wave_on ? quotient(wave_row, a.by_group) : 0;
        const int wave_i1 = wave_on ? quotient(wave_end - 1, a.by_group) : 0;
        const int any_first = row_first(a, rq, wave_i0), any_last = wave_on ? row_last(a, rq, wave_i1) : 0;
        const int all_first = row_first(a, rq, wave_i1), all_last = row_last(a, rq, wave_i0);
        bool row_on[2];
        int i_row[2], q_head[2], last_n[2], first_n[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = wave_row + 16 * r + n;
            row_on[r] = row < rows;
            i_row[r] = row_on[r] ? quotient(row, a.by_group) : wave_i1;
            q_head[r] = head * group + (row_on[r] ? int(row) - i_row[r] * group : 0);
            last_n[r] = row_last(a, rq, i_row[r]);
            first_n[r] = row_first(a, rq, i_row[r]);
        }

        // bf16: the row's query times the scale and log2(e), rounded to fp16's 11 bits, so that a product is an exponent.
        // fp16's range takes it where the largest element is from 2^-6 to below 2^14 (what is lost below 2^-25 is 2^-19
        // of that element or less). Other rows are brought to 2^10 by a power of two, and the products are multiplied by
        // `back`; so are those of fp32 and fp16 queries, without the scale, so that they keep their bits.
        constexpr bool kRaw = S::kExact;
        f16x8 q[S::kQ][2][NB];
        float back[2] = {1.0f, 1.0f};
        bool plain = true;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const T *src = static_cast<const T *>(a.q) + int64_t(rq.begin + i_row[r]) * a.q_stride + int64_t(q_head[r]) * D;
            f32x8 x[NB];
            float mag = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                x[b] = load8(src + 32 * b + 8 * g);
#pragma unroll
                for (int e = 0; e < 8; ++e) mag = fmaxf(mag, fabsf(x[b][e]));
            }
            mag = fmaxf(mag, xor_shfl<16>(mag));
            mag = fmaxf(mag, xor_shfl<32>(mag));
            float factor = a.scale_log2;
            if constexpr (!kRaw) mag *= fabsf(a.scale_log2);
            const bool fits = !kRaw && (mag == 0.0f || (mag >= 0x1p-6f && mag < 0x1p14f));
            plain = plain && __all(fits || !row_on[r]);
            if (!fits) {
                const int exponent = mag > 0.0f && mag < INFINITY ? max(-110, ilogbf(mag)) : 10;
                factor = ldexpf(kRaw ? 1.0f : a.scale_log2, 10 - exponent);
                back[r] = ldexpf(kRaw ? a.scale_log2 : 1.0f, exponent - 10);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = x[b][e] * factor;
                    q[0][r][b][e] = (_Float16)v;
                    if constexpr (S::kQ == 2) q[1][r][b][e] = (_Float16)(v - (float)q[0][r][b][e]);
                }
        }

        // ---- into LDS --------------------------------------------------------
        auto bits = [](f16x2 x) { return __builtin_bit_cast(uint32_t, x); };
        const uint32_t magic = magic_bits();
        auto pair_of = [&](uint32_t w) { return __builtin_bit_cast(f16x2, low_numbers(w, magic)); };
        auto high_pair_of = [&](uint32_t w) { return __builtin_bit_cast(f16x2, high_numbers(w, magic)); };
        // N products of two at `to`, and what their rounding left at the second part
        auto put = [&](uint8_t *to, auto count, const f16x2 *v, const f16x2 *d) {
            constexpr int N = decltype(count)::value;
            uint32_t hi[N], lo[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const f16x2 r = v[i] * d[i];
                hi[i] = bits(r);
                if constexpr (S::kParts == 2) lo[i] = bits(__builtin_elementwise_fma(v[i], d[i], -r));
            }
            auto write = [](uint8_t *at, const uint32_t *x) {
                if constexpr (N == 4) *reinterpret_cast<uint4 *>(at) = uint4{x[0], x[1], x[2], x[3]};
                else if constexpr (N == 2) *reinterpret_cast<uint2 *>(at) = uint2{x[0], x[1]};
                else *reinterpret_cast<uint32_t *>(at) = x[0];
            };
            write(to, hi);
            if constexpr (S::kParts == 2) write(to + S::kPart, lo);
        };
        auto decode_piece = [&](Incoming in, int u, int step) __attribute__((always_inline)) {
            uint8_t *buffer = lds + (step & 1) * S::kBuffer;
            const int my_token = token_of(u);
            constexpr int kKeyScales = NB == 2 ? 1 : 2;
            uint32_t big = 0;  // bit t: the piece's token t is divided by 8 (keys: a piece is of one token)
            // of keys not before here: looked at where the tile is loaded, it would be waited for there
            const uint32_t check = !keys ? in.check : NB > 2 && (piece / (NB > 2 ? NB / 4 : 1)) & 1 ? in.scale[1] : in.scale[0];
            if (__any(!in.page_ok || large_scale(check))) {
                const int scales = keys ? 2 * kKeyScales : 16;
                auto token_at = [&](int i) { return keys ? 0 : i / NB; };
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i < scales) {
                        const int e = exponent_of(in.scale[i / 2] >> (16 * (i & 1)));
                        big |= uint32_t(e >= 28 && e < 31) << token_at(i);
                    }
                if constexpr (NB == 8)  // the scales of a key are between two lanes
                    if (keys) big |= (uint32_t)xor_shfl<S::kRowLanes>((int)big);
                if (lane == 0) marked[step & 1] = step;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i < scales) {
                        f16x2 two = __builtin_bit_cast(f16x2, in.scale[i / 2]);
                        if (big >> token_at(i) & 1) two[i & 1] = two[i & 1] * (_Float16)0.125f;
                        if (!keys && exponent_of(in.scale[i / 2] >> (16 * (i & 1))) == 31) two[i & 1] = (_Float16)0.0f;
                        in.scale[i / 2] = __builtin_bit_cast(uint32_t, two);
                    }
            }
            if (keys) {
                if (lane < S::kRowLanes) score_more[step & 1][my_token] = big ? 7.0f : 0.0f;
            } else {
                if (c < S::kChunkTokens) value_shift[step & 1][my_token + c] = big >> c & 1 ? 3.0f : 0.0f;
            }
            if (keys) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int word = piece * 4 + i, slice = word / NB, b = word % NB;
                    const int at = NB == 2 ? i & 1 : i;
                    const f16x2 two = __builtin_bit_cast(f16x2, in.scale[at / 2]);
                    const f16x2 d1 = {two[at & 1], two[at & 1]}, d[4] = {d1, d1, d1, d1};
                    const uint32_t w = in.w[i];
                    const f16x2 v[4] = {pair_of(w), high_pair_of(w), pair_of(w >> 8), high_pair_of(w >> 8)};
                    put(buffer + ((my_token / 16 * NB + b) * 64 + 16 * slice + my_token % 16) * 16,
                        std::integral_constant<int, 4>(), v, d);
                }
            } else {
                // by four tokens (two at D = 256): the lane group that takes them has them in half of its 16 bytes
                constexpr int kPairs = S::kChunkTokens >= 4 ? 2 : 1, kParts4 = S::kChunkTokens / 2 / kPairs;
#pragma unroll
                for (int f = 0; f < kParts4; ++f) {
                    const int t4 = my_token + 4 * f;
                    uint8_t *values = buffer + S::kParts * S::kPart +
                                      ((t4 / 32 * kDepth * 64) + 16 * (t4 / 4 % 4) + c) * 16 + t4 / 16 % 2 * 8 +
                                      (kPairs == 1 ? t4 / 2 % 2 * 4 : 0);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        f16x2 lo[kPairs], hi[kPairs], d[kPairs];
#pragma unroll
                        for (int i = 0; i < kPairs; ++i) {
                            // byte b and scale b of two tokens
                            const int t0 = (4 * f + 2 * i) * NB + b, t1 = t0 + NB;
                            const uint32_t pair = __builtin_amdgcn_perm(in.w[t1 / 4], in.w[t0 / 4],
                                                                        0x0c000c00u | ((4u + t1 % 4) << 16) | (t0 % 4));
                            lo[i] = pair_of(pair);
                            hi[i] = high_pair_of(pair);
                            const uint32_t s0 = 2 * (t0 & 1), s1 = 4 + 2 * (t1 & 1);
                            d[i] = __builtin_bit_cast(
                                f16x2, __builtin_amdgcn_perm(in.scale[t1 / 2], in.scale[t0 / 2],
                                                             s0 | ((s0 + 1) << 8) | (s1 << 16) | ((s1 + 1) << 24)));
                        }
                        put(values + 2 * b * 1024, std::integral_constant<int, kPairs>(), lo, d);
                        put(values + 2 * b * 1024 + 1024, std::integral_constant<int, kPairs>(), hi, d);
                    }
                }
            }
        };
        auto decode = [&](const Tile &tile, int step) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < S::kPieces; ++u) decode_piece(tile.piece[u], u, step);
        };

        // ---- the rows --------------------------------------------------------
        f32x4 o[2][kDepth] = {};
        // Probabilities are 2^(score - base) with a whole number for base, so that moving it is exact. The products of
        // a plain wave start from -base and end as those exponents (bf16 results: the sums are then rounded at the
        // size of base).
        float base[2] = {0.0f, 0.0f}, l[2] = {0.0f, 0.0f};
        float limit[2] = {-INFINITY, -INFINITY};  // base moves when an exponent is above: at the first one, then at 15
        f32x4 minus_base[2] = {};
        uint32_t broken[2] = {0, 0};  // blocks of the row that are NaN

        // of a marked tile's token: bit 0 no page, bit 1 + b block b of its values is NaN
        auto look_at = [&](int key) -> uint32_t {
            const int page = table[min(key >> a.page_shift, a.max_pages - 1)], token = key & (a.page_size - 1);
            if ((uint32_t)page >= (uint64_t)a.pages) return 1u;
            const uint8_t *p = cache + int64_t(page) * 2 * half_bytes + half_bytes + kv_scale(a.page_size, token, 0, D);
            uint32_t f = 0;
            for (int b = 0; b < NB; ++b)
                if (exponent_of(reinterpret_cast<const uint16_t *>(p)[b]) == 31) f |= 2u << b;
            return f;
        };

        // Of the two waves of a SIMD, which is served first: one that is behind its scores (one part), or before its products
        // with the values (two parts). Without: 1024 new tokens of 16384, 24 heads of 64, bf16 156 us, with it 147; 32 heads
        // over 8 of 128, fp32 580 and 548, fp16 505 and 480, bf16 the same. Both ways round for each were measured, and
        // each stretch alone.
        auto before_scores = [&]() __attribute__((always_inline)) { if constexpr (W == 8 && S::kExact) __builtin_amdgcn_s_setprio(1); };
        auto behind_scores = [&]() __attribute__((always_inline)) { if constexpr (W == 8 && !S::kExact) __builtin_amdgcn_s_setprio(1); };
        auto before_values = [&]() __attribute__((always_inline)) { if constexpr (W == 8 && S::kExact) __builtin_amdgcn_s_setprio(0); };
        auto behind_values = [&]() __attribute__((always_inline)) { if constexpr (W == 8 && !S::kExact) __builtin_amdgcn_s_setprio(0); };
        // kPass tiles of 16 keys, from tile t0 of the step's on
        auto multiply_pass = [&](int step, int t0) __attribute__((always_inline)) {
            const uint8_t *key_operands = lds + (step & 1) * S::kBuffer + t0 * NB * 1024 + lane * 16;
            const uint8_t *value_operands =
                lds + (step & 1) * S::kBuffer + S::kParts * S::kPart + t0 / 2 * kDepth * 1024 + lane * 16;
            // of tile t's keys that this lane has: at 16 t
            const float *more = &score_more[step & 1][16 * t0 + 4 * g], *shifts = &value_shift[step & 1][16 * t0 + 4 * g];
            const int key0 = key_lo + step * KT + 16 * t0;
            if (key0 >= any_last || key0 + 16 * kPass <= any_first) return;
            const bool whole = key0 >= all_first && key0 + 16 * kPass <= all_last;
            const bool odd = marked[step & 1] == step;
            f32x4 s[2][kPass];  // tile t: keys 16t + 4g + 0..3
            {
                constexpr int kReads = kPass * NB * S::kParts;
                before_scores();
                auto read = [&](int r) {
                    return *reinterpret_cast<const f16x8 *>(key_operands + r / S::kParts * 1024 + r % S::kParts * S::kPart);
                };
                f16x8 ring[kAhead];
#pragma unroll
                for (int r = 0; r < kAhead; ++r) ring[r] = read(r);
                pin_order();
#pragma unroll
                for (int r = 0; r < kReads; ++r) {
                    const int t = r / S::kParts / NB, b = r / S::kParts % NB;
                    const f16x8 k = ring[r % kAhead];
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        if (r % (NB * S::kParts) == 0) s[w][t] = minus_base[w];
                        s[w][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[0][w][b], s[w][t], 0, 0, 0);
                    }
                    if constexpr (S::kQ == 2)
                        if (r % S::kParts == 0)
#pragma unroll
                            for (int w = 0; w < 2; ++w)
                                s[w][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[1][w][b], s[w][t], 0, 0, 0);
                    if (r + kAhead < kReads) ring[r % kAhead] = read(r + kAhead);
                    pin_order();
                }
            }
            behind_scores();
            // the first values are on their way while the exponents are looked at
            constexpr int kValueReads = kPass / 2 * kDepth * S::kParts;
            auto read_values = [&](int r) {
                return *reinterpret_cast<const f16x8 *>(value_operands + r / S::kParts * 1024 + r % S::kParts * S::kPart);
            };
            f16x8 ring[kAhead];
#pragma unroll
            for (int r = 0; r < kAhead; ++r) ring[r] = read_values(r);
            auto key_of = [&](int t, int i) { return key0 + 16 * t + 4 * g + i; };
            if (odd) {
                // of what the scores are without the base
#pragma unroll
                for (int t = 0; t < kPass; ++t) {
                    const f32x4 times = *reinterpret_cast<const f32x4 *>(more + 16 * t);
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float within = kRaw || !plain ? 0.0f : base[w];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[w][t][i] = __builtin_fmaf(s[w][t][i] + within, times[i], s[w][t][i]);
                    }
                    pin_order();
                }
            }
            if (kRaw || !plain) {
#pragma unroll
                for (int t = 0; t < kPass; ++t)
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[w][t][i] = __builtin_fmaf(s[w][t][i], back[w], -base[w]);
            }
            if (!whole || odd) {
                uint32_t hidden = 0;  // one bit for each of the lane's keys
                if (odd) {
#pragma unroll 1
                    for (int i = 0; i < 4 * kPass; ++i) {
                        const int key = key_of(i / 4, i % 4);
                        const uint32_t f = look_at(key);
                        hidden |= (f & 1u) << i;
                        for (int w = 0; w < 2; ++w)
                            if (!(f & 1u) && key >= first_n[w] && key < last_n[w]) broken[w] |= f >> 1;
                    }
                }
#pragma unroll
                for (int t = 0; t < kPass; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key_of(t, i);
                        const bool there = !(hidden >> (4 * t + i) & 1u);
#pragma unroll
                        for (int w = 0; w < 2; ++w)
                            s[w][t][i] = there && key >= first_n[w] && key < last_n[w] ? s[w][t][i] : -INFINITY;
                    }
            }
            // The base is taken so that the largest probability is 2^12, and moves to a larger score only once that
            // is 3 above: up to 2^15 fp16 still holds them, and a row's largest scores come early. A tile with values
            // divided by 8 uses those 3 itself and moves at once. (Past 2^24 the base itself is rounded, to what fp32
            // tells apart of the scores. Past 2^26 x - 12 is x - 16, then x: the largest probability is cut to what fp16
            // holds, or is 1.)
            float mx[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                mx[w] = s[w][0][0];
#pragma unroll
                for (int t = 0; t < kPass; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx[w] = __builtin_elementwise_maximum(mx[w], s[w][t][i]);
            }
            const float most = odd ? 12.0f : 15.0f;
            // whether a row's base has to move shows in any of its four lanes
            if (__any(mx[0] > fminf(limit[0], most) || mx[1] > fminf(limit[1], most))) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    float x = mx[w];
                    x = __builtin_elementwise_maximum(x, xor_shfl<16>(x));
                    x = __builtin_elementwise_maximum(x, xor_shfl<32>(x));
                    const bool first = limit[w] == -INFINITY;
                    const float by = x > (first ? -INFINITY : 12.0f) ? rintf(x - 12.0f) : 0.0f;
                    if (x > -INFINITY) limit[w] = 15.0f;
                    const float alpha = first ? 1.0f : exp2_of(-by);
                    base[w] += by;
                    l[w] *= alpha;
#pragma unroll
                    for (int t = 0; t < kDepth; ++t) o[w][t] *= alpha;
#pragma unroll
                    for (int t = 0; t < kPass; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[w][t][i] = __builtin_elementwise_minimum(s[w][t][i] - by, most + 0.5f);
                    if (!kRaw && plain) minus_base[w] = f32x4{-base[w], -base[w], -base[w], -base[w]};
                }
            }
            if (odd) {
                // probabilities of divided values are 8 times as large, and enter the sum as they are: 7/8 of them leave it
#pragma unroll
                for (int t = 0; t < kPass; ++t) {
                    const f32x4 shift = *reinterpret_cast<const f32x4 *>(shifts + 16 * t);
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (shift[i] != 0.0f) {
                                const float p = exp2_of(s[w][t][i] += shift[i]);
                                l[w] -= 0.875f * (S::kParts == 1 ? (float)(_Float16)p : p);
                            }
                    pin_order();
                }
            }
            // Probabilities of 8 keys a lane at a time, of two tiles; the next ones between the products with these.
            f16x8 p0[2][2], p1[2][2];
            float sum[2] = {0.0f, 0.0f};
            auto probabilities = [&](int c2, int w, int e) __attribute__((always_inline)) {  // two of the 32 keys c2's, from slot e on
                const int t = 2 * c2 + e / 4;
#pragma unroll
                for (int i = e; i < e + 2; ++i) {
                    const float p = exp2_of(s[w][t][i % 4]);
                    p0[c2 & 1][w][i] = (_Float16)p;
                    if constexpr (S::kParts == 2) {
                        p1[c2 & 1][w][i] = (_Float16)(p - (float)p0[c2 & 1][w][i]);
                        sum[w] += p;
                    }
                }
                if constexpr (S::kParts == 1) {  // the sum of what is multiplied: of the rounded probabilities
                    const _Float16 one = (_Float16)1.0f;
                    sum[w] = __builtin_amdgcn_fdot2((f16x2){p0[c2 & 1][w][e], p0[c2 & 1][w][e + 1]}, (f16x2){one, one},
                                                    sum[w], false);
                }
            };
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int e = 0; e < 8; e += 2) probabilities(0, w, e);
            pin_order();
            before_values();
#pragma unroll
            for (int r = 0; r < kValueReads; ++r) {
                const int c2 = r / S::kParts / kDepth, t = r / S::kParts % kDepth;
                const f16x8 v = ring[r % kAhead];
#pragma unroll
                for (int w = 0; w < 2; ++w) o[w][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p0[c2 & 1][w], o[w][t], 0, 0, 0);
                if constexpr (S::kParts == 2)
                    if (r % 2 == 0)
#pragma unroll
                        for (int w = 0; w < 2; ++w)
                            o[w][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p1[c2 & 1][w], o[w][t], 0, 0, 0);
                if (r + kAhead < kValueReads) ring[r % kAhead] = read_values(r + kAhead);
                // 8 pairs over the first of the kDepth products
                if (c2 + 1 < kPass / 2 && r % S::kParts == 0) {
                    constexpr int kEach = kDepth >= 8 ? 1 : 8 / kDepth;
#pragma unroll
                    for (int j = t * kEach; j < t * kEach + kEach; ++j)
                        if (j < 8) probabilities(c2 + 1, j & 1, j / 2 * 2);
                }
                pin_order();
            }
            behind_values();
            l[0] += sum[0];
            l[1] += sum[1];
        };
        auto multiply = [&](int step) __attribute__((always_inline)) {
            if constexpr (kSub == kPass) {
                multiply_pass(step, 0);
            } else {
#pragma unroll 1
                for (int t0 = 0; t0 < kSub; t0 += kPass) multiply_pass(step, t0);
            }
        };

        if (step0 < step1) {
            decode(in, step0);
            in = load(step0 + 1, page);
            page = pages_of(step0 + 2);
            __syncthreads();
            auto next = [&](int step) __attribute__((always_inline)) {
                if (step + 1 >= step1) return;
                decode(in, step + 1);
                in = load(step + 2, page);
                page = pages_of(step + 3);
            };
            for (int step = step0; step < step1; ++step) {
                // Each SIMD has a wave that decodes keys and one that decodes values: the one decodes while the other
                // multiplies.
                if (keys) next(step);
                multiply(step);
                if (!keys) next(step);
                __syncthreads();
            }
        }

        // ---- results ---------------------------------------------------------
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float total = l[w] + xor_shfl<16>(l[w]);
            total += xor_shfl<32>(total);
            int nan_blocks = (int)broken[w];
            nan_blocks |= xor_shfl<16>(nan_blocks);
            nan_blocks |= xor_shfl<32>(nan_blocks);
            if (!row_on[w]) continue;
            const int token = rq.begin + i_row[w];
            const int64_t out_at = int64_t(token) * a.q_heads + q_head[w];
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int t = 0; t < kDepth; ++t) {
                const int d = 16 * t + 4 * g;
                f32x4 v = o[w][t];
                if (nan_blocks >> (t / 2) & 1) v += __builtin_nanf("");
                if (used > 1) *reinterpret_cast<f32x4 *>(a.part_out + (out_at * a.splits + split) * D + d) = v;
                else store4(static_cast<T *>(a.out) + token * a.out_stride + int64_t(q_head[w]) * D + d,
                            total == 0.0f ? f32x4{} : v * inv);
            }
            if (g == 0 && a.splits > 1) {
                if (used > 1) {
                    a.part_ml[(out_at * a.splits + split) * 2] = total == 0.0f ? -INFINITY : base[w];
                    a.part_ml[(out_at * a.splits + split) * 2 + 1] = total;
                }
                if (split == 0) a.part_count[out_at] = used;
            }
        }
        if (tid < 2) marked[tid] = -1;  // steps count from the tile's own first key
        __syncthreads();
    }
}

template <int D, class T>
hipError_t launch_typed(const AttendArgs &a, hipStream_t s) {
    constexpr int W = prompt_tile_rows(D) / 32, KT = prompt_tile_keys(D);
    using S = PromptShape<D, T, W, KT>;
    const int64_t grid = int64_t(a.requests) * a.tiles * a.parts * a.kv_heads;
    attention_kv4_prompt_kernel<D, T, W, KT><<<dim3((unsigned)grid), 64 * W, 2 * S::kBuffer, s>>>(a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const AttendArgs &a, int type, hipStream_t s) {
    switch (type) {
    case 0: return launch_typed<D, float>(a, s);
    case 1: return launch_typed<D, __bf16>(a, s);
    default: return launch_typed<D, _Float16>(a, s);
    }
}

}  // namespace

hipError_t launch_attention_kv4_prompt(const AttendArgs &a, int type, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 64: return launch_dim<64>(a, type, s);
    case 128: return launch_dim<128>(a, type, s);
    default: return launch_dim<256>(a, type, s);
    }
}

}  // namespace pfng
