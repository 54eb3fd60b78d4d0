// The paged 4-bit cache: block tables and slots of a step, rows stored as q4_0
// blocks and read back. The cache's format is in kv_layout.h.
#include "io_types.h"
#include "kv_kernels.h"
#include "kv_layout.h"

namespace pfng {
namespace {

// ---------------------------------------------------------------------------
// block tables
// ---------------------------------------------------------------------------
//
//   starts = exclusive sums of added, lengths = cached + added
//   first = ceil(cached / P), end = ceil(length / P), before = exclusive sums of (end - first)
//   table[r, j] = free[before_r + j - first_r] for first <= j < end
//   token i of r: position cached + i, slot table[r, position / P] * P + position % P
//
// A few thousand integers: what counts is the latency of one launch. Every
// workgroup takes the sums over all requests by itself (at most 32 KB from L2)
// and then writes its share of the tokens and requests, so that no workgroup
// waits for another. A token's page comes from the free list or from an entry
// of the table that no workgroup writes. 4 requests 2.5 us, 1000 with
// prompts among them 5.7, where an empty launch takes 2.1.
constexpr int kTablesThreads = 256;

// A count as it is used: the sum of two and a page stays an int.
__device__ __forceinline__ int count_of(int v) { return min(max(v, 0), (1 << 30) - 2048); }

__global__ __launch_bounds__(kTablesThreads) void kv_block_tables_kernel(KvTablesArgs a) {
    extern __shared__ int lds[];  // starts[requests], before[requests], two sums of each wave
    int *starts = lds, *before = lds + a.requests, *sums = before + a.requests;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.requests + kTablesThreads - 1) / kTablesThreads;
    const int r0 = min(tid * per, a.requests), r1 = min(r0 + per, a.requests);
    const int up = a.page_size - 1, shift = a.page_shift;

    int tokens = 0, pages = 0;
    for (int r = r0; r < r1; ++r) {
        const int c = count_of(a.cached[r]), n = count_of(a.added[r]);
        starts[r] = tokens;
        before[r] = pages;
        tokens += n;
        pages += ((c + n + up) >> shift) - ((c + up) >> shift);
    }
    int t_sum = tokens, p_sum = pages;  // inclusive over the wave
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(t_sum, o, 64), p = __shfl_up(p_sum, o, 64);
        if (lane >= o) {
            t_sum += t;
            p_sum += p;
        }
    }
    if (lane == 63) {
        sums[wave] = t_sum;
        sums[4 + wave] = p_sum;
    }
    __syncthreads();
    int t_base = t_sum - tokens, p_base = p_sum - pages;
    for (int w = 0; w < wave; ++w) {
        t_base += sums[w];
        p_base += sums[4 + w];
    }
    for (int r = r0; r < r1; ++r) {
        starts[r] += t_base;
        before[r] += p_base;
    }
    const int total = sums[0] + sums[1] + sums[2] + sums[3];
    __syncthreads();

    if (blockIdx.x == 0 && tid == 0) {
        a.starts[a.requests] = total;
        *a.used = sums[4] + sums[5] + sums[6] + sums[7];
    }
    // requests: one wave each
    for (int r = blockIdx.x * 4 + wave; r < a.requests; r += gridDim.x * 4) {
        const int c = count_of(a.cached[r]), n = count_of(a.added[r]);
        if (lane == 0) {
            a.starts[r] = starts[r];
            a.lengths[r] = c + n;
        }
        const int first = (c + up) >> shift, end = min((c + n + up) >> shift, a.max_pages);
        for (int j = first + lane; j < end; j += 64) {
            const int64_t at = int64_t(before[r]) + (j - first);
            a.table[r * a.table_stride + j] = uint64_t(at) < uint64_t(a.free_count) ? a.free_pages[at] : -1;
        }
    }
    // tokens (sums over the requests that pass 2^31 give wrong places, but none outside the lists)
    for (int64_t t = int64_t(blockIdx.x) * kTablesThreads + tid; t < a.tokens; t += int64_t(gridDim.x) * kTablesThreads) {
        int position = 0, slot = -1;
        if (t < total) {
            int lo = 0, hi = a.requests;  // the last request that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (starts[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int c = count_of(a.cached[lo]);
            position = c + int(min(max(t - starts[lo], int64_t(0)), int64_t(count_of(a.added[lo]))));
            const int j = position >> shift, first = (c + up) >> shift;
            int page = -1;
            if (j < a.max_pages) {
                const int64_t at = int64_t(before[lo]) + (j - first);
                if (j < first) page = a.table[lo * a.table_stride + j];
                else if (uint64_t(at) < uint64_t(a.free_count)) page = a.free_pages[at];
            }
            if (page >= 0 && page <= (INT32_MAX >> shift)) slot = (page << shift) + (position & up);
        }
        a.positions[t] = position;
        a.slots[t] = slot;
    }
}

// ---------------------------------------------------------------------------
// rows into the cache and back
// ---------------------------------------------------------------------------
//
// q4_0 of a block of 32: m the value of largest magnitude (the first of equals),
// d = m / -8, code = min(15, trunc(x / d + 8.5)) with the reciprocal in fp32,
// scale fp16(d): the bytes of pfng_hip_quantize_q4_0 in this cache's places. A
// block that holds an infinity or a NaN gets the scale NaN, so that it reads back
// as NaN and a fault upstream shows.
//
// HBM-bound. Eight elements a lane: D / 8 lanes a row, four a block, and a
// workgroup takes 2048 / D neighbouring tokens of one head, keys and values (both
// by one thread: 15.2 -> 13.0 us). 2048 tokens of 32 heads of 128: stored from bf16
// in 13.1 us, 3.3 TB/s, read to fp32 in 17.7, 4.3 TB/s.
constexpr int kRowThreads = 256;

template <int D>
struct RowShape {
    static constexpr int kLanes = D / 8, kTokens = kRowThreads / kLanes, kBlocks = D / 32;
};

// Code of x in a block with reciprocal scale `id`, clamped to 0..15 also where
// x * id is not finite (a subnormal d).
__device__ __forceinline__ uint32_t q4_code(float x, float id) {
    const int q = (int)add_rn(mul_rn(x, id), 8.5f);
    return (uint32_t)min(15, max(0, q));
}

// The eight codes of a lane, element i at nibble i, and the scale of its block, whose four lanes are neighbours.
struct Coded {
    uint32_t word, scale;
};
__device__ __forceinline__ Coded encode(const f32x8 &x, int j) {
    float top = x[0], mag = fabsf(x[0]);
    int bad = !(mag < INFINITY);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        const float m = fabsf(x[i]);
        bad |= !(m < INFINITY);
        if (m > mag) {
            mag = m;
            top = x[i];
        }
    }
    // the block's value of largest magnitude, the first of equals
    auto meet = [&](float m, float v, bool after) {
        if (m > mag || (m == mag && after)) {
            mag = m;
            top = v;
        }
    };
    meet(xor_shfl<1>(mag), xor_shfl<1>(top), j & 1);
    meet(xor_shfl<2>(mag), xor_shfl<2>(top), j & 2);
    bad |= xor_shfl<1>(bad);
    bad |= xor_shfl<2>(bad);
    const float d = top / -8.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    Coded c = {0, bad ? 0x7e00u : f32_to_fp16_bits(d)};
#pragma unroll
    for (int i = 0; i < 8; ++i) c.word |= (bad ? 8u : q4_code(x[i], id)) << (4 * i);
    return c;
}

template <int D, class T>
__global__ __launch_bounds__(kRowThreads) void kv4_store_kernel(KvRowsArgs a) {
    using S = RowShape<D>;
    __shared__ uint8_t bytes[S::kTokens][D / 2];
    const int tid = threadIdx.x, j = tid % S::kLanes, row = tid / S::kLanes;
    const int head = blockIdx.x % a.kv_heads;
    const int64_t t = int64_t(blockIdx.x / a.kv_heads) * S::kTokens + row;
    const int slot = t < a.tokens ? a.slots[t] : -1;
    const bool on = slot >= 0 && slot < a.slot_count;
    f32x8 k = {}, v = {};
    if (on) {
        k = load8(static_cast<const T *>(a.k) + t * a.k_stride + int64_t(head) * D + j * 8);
        v = load8(static_cast<const T *>(a.v) + t * a.v_stride + int64_t(head) * D + j * 8);
    }
    const Coded kc = encode(k, j), vc = encode(v, j);
    {
        // lanes 4b, 4b + 1 hold nibble 2b of lanes c = 0..7 and 8..15, lanes 4b + 2, 4b + 3 nibble 2b + 1
        const uint32_t other = (uint32_t)xor_shfl<2>((int)vc.word);
        const uint32_t low = (j & 2) ? other : vc.word, high = (j & 2) ? vc.word : other;
        const int b = j >> 2, c0 = 8 * (j & 1) + 2 * (j & 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = 4 * (c0 % 8 + i);
            bytes[row][(c0 + i) * S::kBlocks + b] = uint8_t(((low >> s) & 15u) | (((high >> s) & 15u) << 4));
        }
    }
    __syncthreads();
    if (!on) return;
    const int page = slot >> a.page_shift, token = slot & (a.page_size - 1);
    const int64_t page_bytes = kv_page_bytes(a.page_size, D);
    uint8_t *keys = a.cache + (int64_t(page) * 2 * a.kv_heads + head) * page_bytes, *values = keys + a.kv_heads * page_bytes;
    uint32_t word = 0;  // the even elements' nibbles, then the odd ones'
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= ((kc.word >> (4 * i)) & 15u) << (4 * kv_key_nibble(i));
    *reinterpret_cast<uint32_t *>(keys + kv_key_word(token, j & 3, j >> 2, D)) = word;
    if constexpr (S::kBlocks == 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint16_t *>(values + kv_value_bytes(token, 2 * j + i, D)) =
                *reinterpret_cast<const uint16_t *>(&bytes[row][4 * j + 2 * i]);
    } else {
        constexpr int kWords = S::kBlocks / 4;
        *reinterpret_cast<uint32_t *>(values + kv_value_bytes(token, j / kWords, D) + 4 * (j % kWords)) =
            *reinterpret_cast<const uint32_t *>(&bytes[row][4 * j]);
    }
    if ((j & 3) == 0) {
        const int at = kv_scale(a.page_size, token, j >> 2, D);
        *reinterpret_cast<uint16_t *>(keys + at) = (uint16_t)kc.scale;
        *reinterpret_cast<uint16_t *>(values + at) = (uint16_t)vc.scale;
    }
}

// (code - 8) * scale of the slots; rows of slots outside the cache are zeros.
template <int D, class T>
__global__ __launch_bounds__(kRowThreads) void kv4_read_kernel(KvReadArgs a) {
    using S = RowShape<D>;
    const int tid = threadIdx.x, j = tid % S::kLanes, row = tid / S::kLanes;
    const int head = blockIdx.x % a.kv_heads;
    const int64_t t = int64_t(blockIdx.x / a.kv_heads) * S::kTokens + row;
    if (t >= a.tokens) return;
    const int slot = a.slots[t];
    f32x8 k = {}, v = {};
    if (slot >= 0 && slot < a.slot_count) {
        const int page = slot >> a.page_shift, token = slot & (a.page_size - 1);
        const int64_t page_bytes = kv_page_bytes(a.page_size, D);
        const uint8_t *keys = a.cache + (int64_t(page) * 2 * a.kv_heads + head) * page_bytes;
        const uint8_t *values = keys + a.kv_heads * page_bytes;
        const int at = kv_scale(a.page_size, token, j >> 2, D);
        const float kd = fp16_to_f32(*reinterpret_cast<const uint16_t *>(keys + at));
        const float vd = fp16_to_f32(*reinterpret_cast<const uint16_t *>(values + at));
        const uint32_t word = *reinterpret_cast<const uint32_t *>(keys + kv_key_word(token, j & 3, j >> 2, D));
        const int n = j >> 1;  // values: elements 16 n + c
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t q = values[kv_value_bytes(token, 8 * (j & 1) + i, D) + n / 2];
            k[i] = float(int((word >> (4 * kv_key_nibble(i))) & 15u) - 8) * kd;
            v[i] = float(int((q >> (4 * (n & 1))) & 15u) - 8) * vd;
        }
    }
    const int64_t to = (t * a.kv_heads + head) * D + j * 8;
    store8(static_cast<T *>(a.k) + to, k);
    store8(static_cast<T *>(a.v) + to, v);
}

template <class F>
hipError_t with_dim(int d, F f) {
    switch (d) {
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    default: return f(std::integral_constant<int, 256>());
    }
}

}  // namespace

hipError_t launch_kv_block_tables(const KvTablesArgs &a, hipStream_t s) {
    const int64_t by_tokens = (a.tokens + kTablesThreads - 1) / kTablesThreads, by_requests = (a.requests + 3) / 4;
    const int64_t grid = std::min<int64_t>(256, std::max<int64_t>(1, std::max(by_tokens, by_requests)));
    kv_block_tables_kernel<<<dim3((unsigned)grid), kTablesThreads, (2 * a.requests + 8) * sizeof(int), s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv4_store(const KvRowsArgs &a, int type, int head_dim, hipStream_t s) {
    return with_dim(head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        const int64_t grid = (a.tokens + RowShape<D>::kTokens - 1) / RowShape<D>::kTokens * a.kv_heads;
        const dim3 g((unsigned)grid);
        switch (type) {
        case 0: kv4_store_kernel<D, float><<<g, kRowThreads, 0, s>>>(a); break;
        case 1: kv4_store_kernel<D, __bf16><<<g, kRowThreads, 0, s>>>(a); break;
        default: kv4_store_kernel<D, _Float16><<<g, kRowThreads, 0, s>>>(a); break;
        }
        return hipGetLastError();
    });
}

hipError_t launch_kv4_read(const KvReadArgs &a, int type, int head_dim, hipStream_t s) {
    return with_dim(head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        const int64_t grid = (a.tokens + RowShape<D>::kTokens - 1) / RowShape<D>::kTokens * a.kv_heads;
        const dim3 g((unsigned)grid);
        switch (type) {
        case 0: kv4_read_kernel<D, float><<<g, kRowThreads, 0, s>>>(a); break;
        case 1: kv4_read_kernel<D, __bf16><<<g, kRowThreads, 0, s>>>(a); break;
        default: kv4_read_kernel<D, _Float16><<<g, kRowThreads, 0, s>>>(a); break;
        }
        return hipGetLastError();
    });
}

}  // namespace pfng
