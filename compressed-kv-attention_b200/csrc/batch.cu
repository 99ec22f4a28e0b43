// batch.cu -- host side of the serving-step operators (kvx_batch_*): argument checks, the cut of an
// attention call into items, scratch, launches.
#include <algorithm>
#include <cmath>
#include <new>

#include "host.cuh"
#include "paged.cuh"
#include "prefix.cuh"

using namespace kvx;

struct kvx_batch_s {
    int max_batch = 0, n_q_heads = 0, n_kv_heads = 0, group = 0, dim = 0, dtype = 0;
    int device = 0, sms = 0;
    int64_t cap_rows = 0;   // partial-state rows of the scratch
    float *acc = nullptr;
    float2 *ml = nullptr;
    int32_t *starts = nullptr;
    int *status = nullptr;
    int wait_us = 1000000;     // limit of a wait inside a kernel
    bool runs_taken = false;   // a call failed between the kernels that use the counter of runs and zero it
    ~kvx_batch_s() {
        cudaFree(acc);
        cudaFree(ml);
        cudaFree(starts);
        cudaFree(status);
    }
};

namespace {

constexpr int kMaxTokens = 1 << 30;   // of a prefix, a tail or a rotation (token arithmetic in 32 bits)
constexpr int kMaxHeads = 1 << 16;
int ceil_div(int64_t a, int64_t b) { return int((a + b - 1) / b); }

// A batch of at most this many rows a KV head streams its prefix like a tail; more rows go through
// the tensor-core kernel.
constexpr int kStreamRows = 8;

// The streaming kernel's share of the device beside the prefix kernel.  A prefix item's tile (64 tokens,
// 128 rows) takes a CTA's room about as long as four streamed tiles of 16 tokens at head dims from 128
// on and eight below (the softmax of 128 rows does not shrink with the head), and tails are taken to be
// half of max_len on average.  64 sequences of up to 1024 tokens behind 32K of 128 dims took 82 us one kernel
// after the other and 70 us sharing.  Shares below kLeastShare or above kMostShare are not worth the cut
// (tails of 2 % and of 80 % of the work took 3 % and 25 % longer sharing; the streaming kernel then
// simply follows), and a coded prefix, whose CTAs take a SM each, shares nothing (32 sequences of up to
// 512 tokens behind 32731 coded ones: 74 us shared, 64 not).
constexpr double kLeastShare = 0.15, kMostShare = 0.6;
double stream_share(int dim, int64_t prefix_tiles, int64_t tail_tiles) {
    const double share = double(tail_tiles) / double(tail_tiles + (dim >= 128 ? 4 : 8) * prefix_tiles);
    return share >= kLeastShare && share <= kMostShare ? share : 0.0;
}

// The cut of a prefix for the tensor-core kernel: tiles an item, such that the work of `lists` (KV head,
// 128 rows) pairs ends soonest when `slots` CTAs run at a time.  In tiles' time an item costs its tiles
// and kItemTiles (its queries, the pipeline's fill and drain, the write of its state), and the combine
// pass kPartTiles for every part of a row.
constexpr double kItemTiles = 5.0, kPartTiles = 0.15;
int prefix_split_tiles(int tiles, int lists, int slots) {
    int best = tiles;
    double least = 1e300;
    for (int splits = 1; splits <= tiles && splits <= std::max(1, 2 * slots / lists); ++splits) {
        const int per = ceil_div(tiles, splits), parts = ceil_div(tiles, per);
        const double cost = ceil_div(int64_t(parts) * lists, slots) * (per + kItemTiles) + kPartTiles * parts;
        if (cost < least) least = cost, best = per;
    }
    return best;
}

// CTAs of the streaming kernel that fill the device.
int stream_ctas(const kvx_batch_s *h) { return (h->dim <= 128 ? 2 : 1) * h->sms; }

// Rows of an upper bound of the scratch an attention call of `batch` sequences takes: at most twice as
// many items as CTAs that run at a time, or one for each list, and a part for each run and each unit.
int64_t scratch_rows(const kvx_batch_s *h, int batch) {
    const int64_t rows = int64_t(batch) * h->group;
    const int64_t tensor = (2 * int64_t(prefix_ctas_per_sm(h->dim, false)) * h->sms + h->n_kv_heads * int64_t(ceil_div(rows, kPrefixRows))) *
                           kPrefixRows;
    const int64_t units = h->n_kv_heads * (int64_t(batch) * ceil_div(h->group, 8) + ceil_div(kStreamRows, 8));
    return tensor + 8 * (int64_t(stream_ctas(h)) * kStreamWarps + units);
}

bool attends(int dim) { return dim == 32 || dim == 64 || dim == 128 || dim == 256; }

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool rows_aligned(const kvx_view &v) {
    return aligned16(v.data) && v.token_stride % 8 == 0 && v.head_stride % 8 == 0;
}

PageSplit page_split(int tokens) {
    PageSplit p{tokens, -1};
    if ((tokens & (tokens - 1)) == 0)
        for (p.shift = 0; (1 << p.shift) < tokens;) ++p.shift;
    return p;
}

int pool_of(const char *who, const kvx_pages *p, PoolDev &out) {
    if (p == nullptr || p->k == nullptr || p->v == nullptr || p->n_pages <= 0 || p->page_tokens <= 0 ||
        p->page_stride < 0 || p->token_stride < 0 || p->head_stride < 0)
        return fail(KVX_ERR_INVALID_ARGUMENT, std::string(who) + ": bad page pools");
    out.k = static_cast<uint16_t *>(p->k);
    out.v = static_cast<uint16_t *>(p->v);
    out.page_stride = p->page_stride;
    out.token_stride = p->token_stride;
    out.head_stride = p->head_stride;
    out.n_pages = p->n_pages;
    out.split = page_split(p->page_tokens);
    return KVX_OK;
}

int rope_of(const char *who, const kvx_batch_s *h, const kvx_rope *r, RotArgs &a) {
    if (r->cos == nullptr || r->sin == nullptr || r->pos == nullptr || r->n_pos <= 0 || r->rot_dim <= 0 ||
        r->rot_dim % 2 != 0 || r->rot_dim > h->dim || r->n_axes <= 0 || r->n_axes > 255 ||
        (r->n_axes > 1 && r->axis == nullptr))
        return fail(KVX_ERR_INVALID_ARGUMENT, std::string(who) + ": bad rotation");
    a.cos = r->cos;
    a.sin = r->sin;
    a.pos = r->pos;
    a.axis = r->axis;
    a.pos_stride = r->pos_stride;
    a.n_pos = r->n_pos;
    a.rot_dim = r->rot_dim;
    a.n_axes = r->n_axes;
    a.interleaved = r->interleaved != 0;
    return KVX_OK;
}

// Whether a launch may take 16 values a thread: every row it reads or writes starts on 16 bytes and
// the rotated part and the rest are whole 16-value pieces.
bool vector_path(const RotArgs &a, int n_seg) {
    if (a.dim % 16 != 0 || a.rot_dim % 16 != 0) return false;
    if (a.rot_dim > 0 && (!aligned16(a.cos) || !aligned16(a.sin) || (reinterpret_cast<uintptr_t>(a.axis) & 7u) != 0))
        return false;
    for (int i = 0; i < n_seg; ++i) {
        const RotSeg &s = a.seg[i];
        if (!aligned16(s.src) || s.src_token % 8 != 0 || s.src_head % 8 != 0) return false;
        if (s.pool == 0 && (!aligned16(s.dst) || s.dst_token % 8 != 0 || s.dst_head % 8 != 0)) return false;
        if (s.pool != 0 && (!aligned16(s.pool == 1 ? a.pool.k : a.pool.v) || a.pool.page_stride % 8 != 0 ||
                            a.pool.token_stride % 8 != 0 || a.pool.head_stride % 8 != 0))
            return false;
    }
    return true;
}

RotSeg seg_of(const kvx_view *src, const kvx_view *dst, int heads, bool rotated, int pool) {
    RotSeg s{};
    s.src = static_cast<const uint16_t *>(src->data);
    s.src_token = src->token_stride;
    s.src_head = src->head_stride;
    if (dst != nullptr) {
        s.dst = static_cast<uint16_t *>(dst->data);
        s.dst_token = dst->token_stride;
        s.dst_head = dst->head_stride;
    }
    s.heads = heads;
    s.rotated = rotated;
    s.pool = pool;
    return s;
}

// Whether the current device is the handle's (its scratch and its kernels' limits are there).
int on_device(const char *who, const kvx_batch_s *h) {
    int dev = 0;
    KVX_CUDA(cudaGetDevice(&dev));
    if (dev == h->device) return KVX_OK;
    return fail(KVX_ERR_INVALID_ARGUMENT, std::string(who) + ": the batch was made on device " + std::to_string(h->device) +
                                              ", and device " + std::to_string(dev) + " is current");
}

int done() {
    clear_error();
    return KVX_OK;
}

bool view_ok(const kvx_view *v) { return v != nullptr && v->data != nullptr; }

}  // namespace

extern "C" {

int kvx_batch_create(int max_batch, int n_q_heads, int n_kv_heads, int dim, int dtype, kvx_batch *out) {
    if (out == nullptr || max_batch <= 0 || max_batch > kMaxStreamBatch || n_q_heads <= 0 || n_q_heads > kMaxHeads ||
        n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || dim <= 0 || dim % 2 != 0 || dim > kMaxHeadDim ||
        (dtype != KVX_DTYPE_BF16 && dtype != KVX_DTYPE_FP16))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_create: bad argument");
    *out = nullptr;
    if (int rc = check_device()) return rc;
    auto *h = new (std::nothrow) kvx_batch_s();
    if (h == nullptr) return fail(KVX_ERR_RUNTIME, "kvx_batch_create: out of host memory");
    h->max_batch = max_batch;
    h->n_q_heads = n_q_heads;
    h->n_kv_heads = n_kv_heads;
    h->group = n_q_heads / n_kv_heads;
    h->dim = dim;
    h->dtype = dtype;
    h->sms = sm_count();
    cudaError_t e = cudaGetDevice(&h->device);
    h->cap_rows = scratch_rows(h, max_batch);
    if (e == cudaSuccess) e = cudaMalloc(&h->status, 2 * sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(h->status, 0, 2 * sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc(&h->starts, (size_t(max_batch) + 2) * sizeof(int32_t));
    if (e == cudaSuccess) e = cudaMemset(h->starts, 0, (size_t(max_batch) + 2) * sizeof(int32_t));
    if (e == cudaSuccess) e = cudaMalloc(&h->acc, size_t(h->cap_rows) * dim * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&h->ml, size_t(h->cap_rows) * sizeof(float2));
    if (e == cudaSuccess && attends(dim)) e = prepare_paged_prefix(dim, dtype);
    if (e == cudaSuccess && attends(dim)) e = prepare_paged_stream(dim, dtype);
    if (e != cudaSuccess) {
        delete h;
        return fail(KVX_ERR_CUDA, std::string("kvx_batch_create: ") + cudaGetErrorString(e));
    }
    *out = h;
    return done();
}

void kvx_batch_destroy(kvx_batch h) { delete h; }

int kvx_batch_check(kvx_batch h) {
    if (h == nullptr) return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_check: null batch");
    if (int rc = on_device("kvx_batch_check", h)) return rc;
    KVX_CUDA(cudaDeviceSynchronize());
    if (int rc = read_status(h->status, true)) return rc;
    return done();
}

int kvx_batch_wait_limit(kvx_batch h, int microseconds) {
    if (h == nullptr || microseconds < 0)
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_wait_limit: bad argument");
    h->wait_us = microseconds;
    return done();
}

int kvx_batch_rotate(kvx_batch h, const kvx_view *x, const kvx_view *out, int n_tokens, int n_heads,
                     const kvx_rope *rope, int inverse, void *stream) {
    if (h != nullptr && n_tokens == 0) return done();  // (an empty tensor's address is null)
    if (h == nullptr || !view_ok(x) || !view_ok(out) || n_tokens < 0 || n_tokens > kMaxTokens || n_heads <= 0 ||
        n_heads > kMaxHeads || rope == nullptr)
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_rotate: bad argument");
    if (int rc = on_device("kvx_batch_rotate", h)) return rc;
    RotArgs a{};
    if (int rc = rope_of("kvx_batch_rotate", h, rope, a)) return rc;
    a.seg[0] = seg_of(x, out, n_heads, true, 0);
    a.inverse = inverse != 0;
    a.status = h->status;
    a.n_tokens = n_tokens;
    a.dim = h->dim;
    a.heads = n_heads;
    KVX_CUDA(launch_rotate(h->dtype, vector_path(a, 1), a, static_cast<cudaStream_t>(stream)));
    return done();
}

int kvx_batch_append(kvx_batch h, const kvx_view *q, const kvx_view *k, const kvx_view *v, const kvx_view *q_out,
                     int n_tokens, const kvx_rope *rope, const int64_t *slots, const kvx_pages *pages, void *stream) {
    if (h != nullptr && n_tokens == 0) return done();
    const bool has_q = q != nullptr && q->data != nullptr;
    if (h == nullptr || !view_ok(k) || !view_ok(v) || n_tokens < 0 || n_tokens > kMaxTokens || slots == nullptr ||
        has_q != (q_out != nullptr && q_out->data != nullptr))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_append: bad argument");
    if (int rc = on_device("kvx_batch_append", h)) return rc;
    RotArgs a{};
    if (int rc = pool_of("kvx_batch_append", pages, a.pool)) return rc;
    if (rope != nullptr)
        if (int rc = rope_of("kvx_batch_append", h, rope, a)) return rc;
    int n = 0;
    if (has_q) a.seg[n++] = seg_of(q, q_out, h->n_q_heads, rope != nullptr, 0);
    a.seg[n++] = seg_of(k, nullptr, h->n_kv_heads, rope != nullptr, 1);
    a.seg[n++] = seg_of(v, nullptr, h->n_kv_heads, false, 2);
    a.slots = slots;
    a.status = h->status;
    a.n_tokens = n_tokens;
    a.dim = h->dim;
    a.heads = (has_q ? h->n_q_heads : 0) + 2 * h->n_kv_heads;
    KVX_CUDA(launch_rotate(h->dtype, vector_path(a, n), a, static_cast<cudaStream_t>(stream)));
    return done();
}

int kvx_batch_attend(kvx_batch h, const kvx_attend *x, void *stream) {
    if (h != nullptr && x != nullptr && x->batch == 0) return done();
    if (h == nullptr || x == nullptr || x->batch < 0 || x->batch > h->max_batch || !view_ok(&x->q) ||
        !view_ok(&x->out) || x->prefix_len < 0 || x->max_len < 0 || x->prefix_len > kMaxTokens ||
        x->max_len > kMaxTokens || !(x->scale >= 0.f))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: bad argument");
    if (int rc = on_device("kvx_batch_attend", h)) return rc;
    if (!attends(h->dim))
        return fail(KVX_ERR_UNSUPPORTED, "kvx_batch_attend: head_dim must be 32, 64, 128 or 256");
    const bool coded = x->prefix != nullptr, paged = !coded && x->prefix_table != nullptr && x->prefix_len > 0;
    if (coded && (x->prefix_table != nullptr || x->prefix_len > 0))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: one prefix, in pages or as blobs");
    if (coded && (h->dtype != KVX_DTYPE_BF16 || x->prefix->dim != h->dim || x->prefix->n_kv_heads != h->n_kv_heads))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: the prefix is BF16 and of other heads or another head_dim");
    if (coded && x->prefix->device != h->device)
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: the prefix is on another device");
    if (!coded && x->prefix_len > 0 && x->prefix_table == nullptr)
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: a prefix without its page table");
    if (x->max_len > 0 && (x->table == nullptr || x->lens == nullptr))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: tails without page table or lengths");
    if (!rows_aligned(x->q))
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: query rows must be 16-byte aligned");
    PagedArgs a{};
    if (int rc = pool_of("kvx_batch_attend", x->pages, a.pool)) return rc;
    if (!aligned16(a.pool.k) || !aligned16(a.pool.v) || a.pool.page_stride % 8 != 0 || a.pool.token_stride % 8 != 0 ||
        a.pool.head_stride % 8 != 0)
        return fail(KVX_ERR_INVALID_ARGUMENT, "kvx_batch_attend: page rows must be 16-byte aligned");
    a.q = static_cast<const uint16_t *>(x->q.data);
    a.q_token = x->q.token_stride;
    a.q_head = x->q.head_stride;
    a.out = static_cast<uint16_t *>(x->out.data);
    a.out_token = x->out.token_stride;
    a.out_head = x->out.head_stride;
    a.lse = x->lse;
    a.prefix_table = x->prefix_table;
    a.table = x->table;
    a.lens = x->lens;
    a.table_stride = x->table_stride;
    a.prefix_len = paged ? x->prefix_len : 0;
    if (coded) a.xkv = x->prefix->dev;
    a.max_len = x->max_len;
    a.batch = x->batch;
    a.n_q_heads = h->n_q_heads;
    a.n_kv_heads = h->n_kv_heads;
    a.group = h->group;
    a.scale_log2 = float((x->scale > 0.f ? double(x->scale) : 1.0 / std::sqrt(double(h->dim))) * 1.4426950408889634);
    a.acc = h->acc;
    a.ml = h->ml;
    a.status = h->status;
    a.wait_us = h->wait_us;
    a.starts = h->starts;
    a.next_run = h->starts + h->max_batch + 1;
    const int rows = x->batch * h->group;
    const bool tensor = coded || (paged && rows > kStreamRows);
    if (tensor) {
        a.row_groups = ceil_div(rows, kPrefixRows);
        a.row_pad = kPrefixRows * a.row_groups;
        a.prefix_tiles = coded ? a.xkv.tiles : ceil_div(x->prefix_len, kPrefixTile);
        const double share = coded ? 0.0 : stream_share(h->dim, int64_t(a.prefix_tiles) * h->n_kv_heads * a.row_groups,
                                          int64_t(x->batch) * h->n_kv_heads * ceil_div(h->group, 8) * ceil_div(x->max_len, 2 * kStreamTile));
        const int slots = prefix_ctas_per_sm(h->dim, coded) * h->sms;
        a.split_tiles = prefix_split_tiles(a.prefix_tiles, h->n_kv_heads * a.row_groups, std::max(1, int(slots * (1.0 - share))));
        a.shared_runs = share > 0.0;
        a.n_split = ceil_div(a.prefix_tiles, a.split_tiles);
        a.stream_base = int64_t(h->n_kv_heads) * a.n_split * a.row_pad;
    }
    a.tail_groups = ceil_div(h->group, 8);
    a.pre_groups = ceil_div(rows, 8);
    if (paged && !tensor) a.stream_prefix = h->n_kv_heads * a.pre_groups;
    const int64_t units = a.stream_prefix + int64_t(x->batch) * h->n_kv_heads * a.tail_groups;
    const int64_t most_tiles = int64_t(a.stream_prefix) * ceil_div(x->prefix_len, kStreamTile) +
                               int64_t(x->batch) * h->n_kv_heads * a.tail_groups * ceil_div(x->max_len, kStreamTile);
    if (most_tiles + units * kUnitTiles > INT32_MAX - (1 << 20))  // (positions are counted in 32 bits)
        return fail(KVX_ERR_UNSUPPORTED, "kvx_batch_attend: more than 2^31 tiles of 16 tokens in one call");
    a.stream_ctas = int(std::min<int64_t>(stream_ctas(h), ceil_div(most_tiles, kStreamWarps)));
    a.stream_runs = a.stream_ctas * kStreamWarps;
    const int64_t used = a.stream_base + (a.stream_ctas > 0 ? 8 * (int64_t(a.stream_runs) + units) : 0);
    if (used > h->cap_rows) return fail(KVX_ERR_RUNTIME, "kvx_batch_attend: scratch too small");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.shared_runs) {
        // the combine pass zeroes the counter: where it was not launched, the streaming kernel would find no runs
        if (h->runs_taken) KVX_CUDA(cudaMemsetAsync(a.next_run, 0, sizeof(int32_t), s));
        h->runs_taken = true;
    }
    if (tensor) KVX_CUDA(launch_paged_prefix(h->dim, h->dtype, a, s));
    KVX_CUDA(launch_paged_stream(h->dim, h->dtype, a, tensor, s));
    KVX_CUDA(launch_paged_combine(h->dim, h->dtype, a, s));
    if (a.shared_runs) h->runs_taken = false;
    return done();
}

}  // extern "C"
