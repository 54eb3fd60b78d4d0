// C-ABI entry points of the serving operators (declared in include/pfng_hip.h):
// the paged 4-bit cache, the norms of query and key heads with the position
// rotation, and attention over the cache. As in api.cpp: arguments are checked on
// the host, launches are asynchronous, nothing throws.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "kv_kernels.h"
#include "kv_layout.h"
#include "pfng_hip.h"
#include "status.h"

namespace {

using pfng::aligned;
using pfng::fail;
using pfng::hip_status;

typedef long long ll;

// Counts above this are refused: positions, keys and slots are 32-bit numbers,
// and sums of two of them stay so.
constexpr int64_t kMost = int64_t(1) << 30;
// Queries' head rows of an attention call, whose workgroups take several row tiles where there are many.
constexpr int64_t kMostRows = int64_t(1) << 32;
// HIP takes fewer than 2^32 threads in a launch: workgroups of 256.
constexpr int64_t kMostGroups = (int64_t(1) << 24) - 1;

int elem_bytes(int type) { return type == PFNG_F32 ? 4 : 2; }

int log2_of(int v) {
    int n = 0;
    while ((1 << n) < v) ++n;
    return n;
}

int check_type(const char *what, int type) {
    if (type < 0 || type > PFNG_F16) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", what, type);
    return PFNG_OK;
}

int check_cache(const char *what, int64_t pages, int kv_heads, int head_dim, int page_size) {
    if (!pfng::kv_head_dim_ok(head_dim))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: head_dim=%d (64, 128 and 256 are supported)", what, head_dim);
    if (!pfng::kv_page_size_ok(page_size))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: page_size=%d must be a power of two from %d to %d", what, page_size,
                    pfng::kKvMinPage, pfng::kKvMaxPage);
    if (kv_heads <= 0 || kv_heads > 65536)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: kv_heads=%d", what, kv_heads);
    if (pages <= 0 || pages > kMost / page_size)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: pages=%lld (1 to %lld pages of %d tokens)", what, (ll)pages,
                    (ll)(kMost / page_size), page_size);
    return PFNG_OK;
}

// Rows of heads x head_dim elements, `stride` elements from token to token.
int check_rows(const char *what, const char *name, const void *p, int64_t stride, int64_t heads, int head_dim, int type) {
    if (!p) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
    if (stride < heads * head_dim || stride > (int64_t(1) << 40))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: %s has a token stride of %lld elements, fewer than its %lld", what,
                    name, (ll)stride, (ll)(heads * head_dim));
    if (!aligned(p, 16) || stride * elem_bytes(type) % 16)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: %s and its rows must be 16-byte aligned", what, name);
    return PFNG_OK;
}

// The kernels that take a row of head_dim elements by head_dim / 8 threads, 2048 elements a workgroup: its workgroups
// where each takes rows of all heads (heads = 1), or of one head.
int check_groups(const char *what, int64_t rows, int64_t heads, int head_dim) {
    const int64_t each = 2048 / head_dim;
    if ((rows + each - 1) / each > kMostGroups / heads)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: %lld rows of %d elements are too many for one launch", what,
                    (ll)(rows * heads), head_dim);
    return PFNG_OK;
}

int current_cus(int *cus) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return fail(PFNG_ERR_HIP, "hipGetDevice failed");
    *cus = pfng::device_cus(dev);
    return PFNG_OK;
}

struct Workspace {
    int64_t out = 0, ml = 0, bytes = 0;  // offsets of the parts' maxima and sums, and of their counts
};

Workspace workspace_of(int64_t tokens, int q_heads, int head_dim, int splits) {
    Workspace w;
    if (splits <= 1) return w;
    const int64_t rows = tokens * q_heads;
    w.out = rows * splits * head_dim * 4;
    w.ml = w.out + rows * splits * 8;
    w.bytes = w.ml + rows * 4;
    return w;
}

int check_attention(int64_t tokens, int64_t requests, int q_heads, int kv_heads, int64_t max_added, int64_t max_length) {
    if (tokens < 0 || tokens > kMost || requests < 0 || requests > kMost)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "attention_kv4: tokens=%lld requests=%lld", (ll)tokens, (ll)requests);
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || q_heads > 65536)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "attention_kv4: q_heads=%d must be a positive multiple of kv_heads=%d",
                    q_heads, kv_heads);
    if (tokens * q_heads > kMostRows || requests * kv_heads > kMostGroups)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "attention_kv4: tokens=%lld requests=%lld heads=%d are too many", (ll)tokens,
                    (ll)requests, q_heads);
    if (tokens * (q_heads / kv_heads) > kMost)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "attention_kv4: %lld tokens of %d heads a key head are too many", (ll)tokens,
                    q_heads / kv_heads);
    if (max_added < 1 || max_added > kMost || max_length < 0 || max_length > kMost)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "attention_kv4: max_added=%lld max_length=%lld", (ll)max_added,
                    (ll)max_length);
    return PFNG_OK;
}

}  // namespace

extern "C" {

int64_t pfng_hip_kv4_page_bytes(int page_size, int head_dim) {
    if (!pfng::kv_head_dim_ok(head_dim) || !pfng::kv_page_size_ok(page_size)) return 0;
    return pfng::kv_page_bytes(page_size, head_dim);
}

int pfng_hip_kv_block_tables(const int32_t *cached, const int32_t *added, int requests, const int32_t *free_pages,
                             int64_t free_count, int page_size, int32_t *block_table, int64_t table_stride,
                             int max_pages, int64_t tokens, int32_t *starts, int32_t *lengths, int32_t *positions,
                             int32_t *slots, int32_t *used, void *stream) {
    if (requests < 0 || requests > pfng::kKvMaxRequests)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "kv_block_tables: requests=%d (0 to %d)", requests, pfng::kKvMaxRequests);
    if (!pfng::kv_page_size_ok(page_size))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "kv_block_tables: page_size=%d must be a power of two from %d to %d",
                    page_size, pfng::kKvMinPage, pfng::kKvMaxPage);
    if (free_count < 0 || tokens < 0 || tokens > kMost)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "kv_block_tables: free_count=%lld tokens=%lld", (ll)free_count, (ll)tokens);
    if (max_pages < 0 || max_pages > kMost / page_size || table_stride < max_pages)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "kv_block_tables: max_pages=%d table_stride=%lld", max_pages,
                    (ll)table_stride);
    if (!starts || !used || (requests && (!cached || !added || !lengths || (max_pages && !block_table))) ||
        (free_count && !free_pages) || (tokens && (!positions || !slots)))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "kv_block_tables: null pointer");
    if (!aligned(cached, 4) || !aligned(added, 4) || !aligned(free_pages, 4) || !aligned(block_table, 4) ||
        !aligned(starts, 4) || !aligned(lengths, 4) || !aligned(positions, 4) || !aligned(slots, 4) || !aligned(used, 4))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "kv_block_tables: pointers must be 4-byte aligned");
    pfng::KvTablesArgs a;
    a.cached = cached, a.added = added, a.free_pages = free_pages;
    a.free_count = free_count, a.tokens = tokens, a.table_stride = table_stride;
    a.table = block_table, a.starts = starts, a.lengths = lengths, a.positions = positions, a.slots = slots;
    a.used = used;
    a.requests = requests, a.max_pages = max_pages, a.page_size = page_size, a.page_shift = log2_of(page_size);
    return hip_status(pfng::launch_kv_block_tables(a, static_cast<hipStream_t>(stream)), "kv_block_tables launch");
}

int pfng_hip_qk_norm_rope(const void *q, int64_t q_stride, const void *k, int64_t k_stride, int in_type, void *q_out,
                          int64_t q_out_stride, void *k_out, int64_t k_out_stride, int out_type, const float *q_weight,
                          const float *k_weight, float eps, const float *cos_sin, int64_t table_rows, int rot_dim,
                          int adjacent, const int32_t *positions, int64_t tokens, int q_heads, int kv_heads,
                          int head_dim, void *stream) {
    const char *what = "qk_norm_rope";
    int rc = check_type(what, in_type);
    if (rc || (rc = check_type(what, out_type))) return rc;
    if (!pfng::kv_head_dim_ok(head_dim))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: head_dim=%d (64, 128 and 256 are supported)", what, head_dim);
    if (tokens < 0 || tokens > kMost || q_heads < 0 || kv_heads < 0 || q_heads > 65536 || kv_heads > 65536)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: tokens=%lld q_heads=%d kv_heads=%d", what, (ll)tokens, q_heads, kv_heads);
    if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 16)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: rot_dim=%d must be a multiple of 16 up to head_dim=%d", what,
                    rot_dim, head_dim);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", what);
    const int64_t rows = tokens * (int64_t(q_heads) + kv_heads);
    if (rows == 0) return PFNG_OK;
    if ((rc = check_groups(what, rows, 1, head_dim))) return rc;
    if (q_heads && ((rc = check_rows(what, "q", q, q_stride, q_heads, head_dim, in_type)) ||
                    (rc = check_rows(what, "q_out", q_out, q_out_stride, q_heads, head_dim, out_type))))
        return rc;
    if (kv_heads && ((rc = check_rows(what, "k", k, k_stride, kv_heads, head_dim, in_type)) ||
                     (rc = check_rows(what, "k_out", k_out, k_out_stride, kv_heads, head_dim, out_type))))
        return rc;
    if (rot_dim && (!cos_sin || table_rows <= 0 || !positions))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: a rotation needs cos_sin, its rows and positions", what);
    if (!aligned(cos_sin, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(positions, 4))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: cos_sin and the weights must be 16-byte, positions 4-byte aligned", what);
    pfng::NormRopeArgs a;
    a.q = q, a.k = k, a.q_stride = q_stride, a.k_stride = k_stride;
    a.q_out = q_out, a.k_out = k_out, a.q_out_stride = q_out_stride, a.k_out_stride = k_out_stride;
    a.q_weight = q_weight, a.k_weight = k_weight, a.cos_sin = cos_sin, a.positions = positions;
    a.tokens = tokens, a.table_rows = table_rows, a.eps = eps;
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.rot_dim = rot_dim, a.adjacent = adjacent != 0;
    return hip_status(pfng::launch_qk_norm_rope(a, in_type, out_type, head_dim, static_cast<hipStream_t>(stream)),
                      "qk_norm_rope launch");
}

int pfng_hip_kv4_store(const void *k, int64_t k_stride, const void *v, int64_t v_stride, int type,
                       const int32_t *slots, int64_t tokens, void *cache, int64_t pages, int kv_heads, int head_dim,
                       int page_size, void *stream) {
    const char *what = "kv4_store";
    int rc = check_type(what, type);
    if (rc || (rc = check_cache(what, pages, kv_heads, head_dim, page_size))) return rc;
    if (tokens < 0 || tokens > kMost) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: tokens=%lld", what, (ll)tokens);
    if (tokens == 0) return PFNG_OK;
    if ((rc = check_groups(what, tokens, kv_heads, head_dim))) return rc;
    if ((rc = check_rows(what, "k", k, k_stride, kv_heads, head_dim, type)) ||
        (rc = check_rows(what, "v", v, v_stride, kv_heads, head_dim, type)))
        return rc;
    if (!slots || !cache) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (!aligned(slots, 4) || !aligned(cache, 16))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: the cache must be 16-byte, slots 4-byte aligned", what);
    pfng::KvRowsArgs a;
    a.k = k, a.v = v, a.k_stride = k_stride, a.v_stride = v_stride, a.slots = slots, a.tokens = tokens;
    a.slot_count = pages * page_size, a.cache = static_cast<uint8_t *>(cache);
    a.kv_heads = kv_heads, a.page_size = page_size, a.page_shift = log2_of(page_size);
    return hip_status(pfng::launch_kv4_store(a, type, head_dim, static_cast<hipStream_t>(stream)), "kv4_store launch");
}

int pfng_hip_kv4_read(const void *cache, int64_t pages, int kv_heads, int head_dim, int page_size,
                      const int32_t *slots, int64_t tokens, void *k, void *v, int type, void *stream) {
    const char *what = "kv4_read";
    int rc = check_type(what, type);
    if (rc || (rc = check_cache(what, pages, kv_heads, head_dim, page_size))) return rc;
    if (tokens < 0 || tokens > kMost) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: tokens=%lld", what, (ll)tokens);
    if (tokens == 0) return PFNG_OK;
    if ((rc = check_groups(what, tokens, kv_heads, head_dim))) return rc;
    if (!slots || !cache || !k || !v) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (!aligned(slots, 4) || !aligned(cache, 16) || !aligned(k, 16) || !aligned(v, 16))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: the cache, k and v must be 16-byte, slots 4-byte aligned", what);
    pfng::KvReadArgs a;
    a.cache = static_cast<const uint8_t *>(cache), a.slots = slots, a.tokens = tokens;
    a.slot_count = pages * page_size, a.k = k, a.v = v;
    a.kv_heads = kv_heads, a.page_size = page_size, a.page_shift = log2_of(page_size);
    return hip_status(pfng::launch_kv4_read(a, type, head_dim, static_cast<hipStream_t>(stream)), "kv4_read launch");
}

int64_t pfng_hip_attention_kv4_workspace_size(int type, int64_t tokens, int64_t requests, int q_heads, int kv_heads,
                                              int head_dim, int causal, int64_t max_added, int64_t max_length) {
    if (check_type("attention_kv4", type)) return -1;
    if (check_attention(tokens, requests, q_heads, kv_heads, max_added, max_length)) return -1;
    if (!pfng::kv_head_dim_ok(head_dim)) {
        fail(PFNG_ERR_INVALID_ARGUMENT, "attention_kv4: head_dim=%d (64, 128 and 256 are supported)", head_dim);
        return -1;
    }
    int cus = 0;
    if (current_cus(&cus)) return -1;
    const pfng::AttendPlan p = pfng::plan_attention(type, tokens, requests, q_heads, kv_heads, head_dim, max_added,
                                                    max_length, causal != 0, cus);
    return workspace_of(tokens, q_heads, head_dim, p.splits).bytes;
}

int pfng_hip_attention_kv4(const void *q, int64_t q_stride, void *out, int64_t out_stride, int type,
                           const int32_t *starts, const int32_t *lengths, int64_t requests, int64_t tokens,
                           int q_heads, const int32_t *block_table, int64_t table_stride, int max_pages,
                           const void *cache, int64_t pages, int kv_heads, int head_dim, int page_size, float scale,
                           int causal, int64_t window, int64_t max_added, int64_t max_length, void *workspace,
                           int64_t workspace_bytes, void *stream) {
    const char *what = "attention_kv4";
    int rc = check_type(what, type);
    if (rc || (rc = check_cache(what, pages, kv_heads, head_dim, page_size)) ||
        (rc = check_attention(tokens, requests, q_heads, kv_heads, max_added, max_length)))
        return rc;
    if (max_pages < 0 || max_pages > kMost / page_size || table_stride < max_pages)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: max_pages=%d table_stride=%lld", what, max_pages, (ll)table_stride);
    if (!std::isfinite(scale)) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: scale must be finite", what);
    if (window < 0) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: window=%lld (0: no window)", what, (ll)window);
    if (!starts && tokens != requests)
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: without starts each request has one token (tokens=%lld requests=%lld)",
                    what, (ll)tokens, (ll)requests);
    if (tokens == 0 || requests == 0) return PFNG_OK;
    if ((rc = check_rows(what, "q", q, q_stride, q_heads, head_dim, type)) ||
        (rc = check_rows(what, "out", out, out_stride, q_heads, head_dim, type)))
        return rc;
    if (!lengths || !cache || (max_pages && !block_table)) return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (!aligned(starts, 4) || !aligned(lengths, 4) || !aligned(block_table, 4) || !aligned(cache, 16))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: the cache must be 16-byte, the other pointers 4-byte aligned", what);
    int cus = 0;
    if ((rc = current_cus(&cus))) return rc;
    const pfng::AttendPlan p = pfng::plan_attention(type, tokens, requests, q_heads, kv_heads, head_dim, max_added,
                                                    max_length, causal != 0, cus);
    const Workspace w = workspace_of(tokens, q_heads, head_dim, p.splits);
    if (w.bytes && (!workspace || workspace_bytes < w.bytes || !aligned(workspace, 16)))
        return fail(PFNG_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld bytes is needed (given: %lld)",
                    what, (ll)w.bytes, workspace ? (ll)workspace_bytes : 0ll);
    pfng::AttendArgs a;
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.starts = starts, a.lengths = lengths, a.table = block_table, a.table_stride = table_stride;
    a.tokens = tokens, a.pages = pages, a.cache = static_cast<const uint8_t *>(cache);
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.requests = (int)requests, a.q_heads = q_heads, a.kv_heads = kv_heads;
    a.max_pages = max_pages, a.page_size = page_size, a.page_shift = log2_of(page_size);
    a.causal = causal != 0, a.window = window < kMost ? (int)window : 0;  // no context is longer
    a.splits = p.splits;
    a.by_group = pfng::Divisor(q_heads / kv_heads), a.by_kv_heads = pfng::Divisor(kv_heads);
    a.by_requests = pfng::Divisor((uint32_t)requests);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    a.part_out = reinterpret_cast<float *>(ws);
    a.part_ml = w.bytes ? reinterpret_cast<float *>(ws + w.out) : nullptr;
    a.part_count = w.bytes ? reinterpret_cast<int32_t *>(ws + w.ml) : nullptr;
    return hip_status(pfng::launch_attention_kv4(a, p, type, head_dim, static_cast<hipStream_t>(stream)), "attention_kv4 launch");
}

}  // extern "C"
