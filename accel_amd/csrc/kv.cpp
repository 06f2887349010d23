// The operator layer's paged key-value cache and attention: argument checks
// and launches (kvpages.hip, attention.hip).  What only the device can see
// (lengths, tables, indices) is checked by the kernels and reported through
// the fault word.
#include <hip/hip_runtime.h>

#include <cmath>

#include "checks.hpp"
#include "internal.hpp"

using namespace accel;

#define ACCEL_API extern "C" __attribute__((visibility("default")))

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The cache as the kernels take it, or a refusal.
int check_cache(const char* op, const accel_kv_cache_t* c, KvCache* out) {
    char buf[256];
    if (!c || !c->keys || !c->values || !c->refs || !c->tables || !c->lens)
        return refuse(op, "the cache needs keys, values, refs, tables and lens");
    if (c->dtype != ACCEL_F16 && c->dtype != ACCEL_BF16) {
        snprintf(buf, sizeof buf, "the cache is %s; keys and values are f16 or bf16",
                 dtype_name(c->dtype));
        return refuse(op, buf);
    }
    if (c->page_size < 8 || c->page_size > 4096 || (c->page_size & (c->page_size - 1))) {
        snprintf(buf, sizeof buf, "pages of %d positions; a page holds a power of two, 8 to 4096",
                 c->page_size);
        return refuse(op, buf);
    }
    if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8) {
        snprintf(buf, sizeof buf, "heads of %d; head_dim is a multiple of 8, 8 to 256",
                 c->head_dim);
        return refuse(op, buf);
    }
    if (c->kv_heads < 1 || c->kv_heads > 4096) {
        snprintf(buf, sizeof buf, "%d key-value heads; 1 to 4096 are served", c->kv_heads);
        return refuse(op, buf);
    }
    if (c->layers < 1 || c->layers > 65535 || c->pages < 1 || c->pages > INT32_MAX ||
        c->sequences < 1 || c->sequences > INT32_MAX || c->slots < 1 || c->slots > INT32_MAX) {
        snprintf(buf, sizeof buf,
                 "a cache of %lld layers, %lld pages, %lld sequences and %lld slots",
                 (long long)c->layers, (long long)c->pages, (long long)c->sequences,
                 (long long)c->slots);
        return refuse(op, buf);
    }
    // positions (with a tile's past the last) and a table's entries are counted
    // in 31 bits
    if (c->slots > (INT32_MAX - 65535) / c->page_size || c->sequences > INT32_MAX / c->slots) {
        snprintf(buf, sizeof buf,
                 "tables of %lld sequences x %lld slots of %d positions are more than 31 bits "
                 "count",
                 (long long)c->sequences, (long long)c->slots, c->page_size);
        return refuse(op, buf);
    }
    // layers * pages * a page's elements stay below 2^62
    const __int128 elems = (__int128)c->layers * c->pages * c->kv_heads * c->page_size *
                           c->head_dim;
    if (elems >= (__int128)1 << 60) return refuse(op, "the cache is larger than an address space");
    if (!aligned16(c->keys) || !aligned16(c->values))
        return refuse(op, "keys and values must start at 16-byte aligned addresses");
    out->keys = static_cast<uint16_t*>(c->keys);
    out->values = static_cast<uint16_t*>(c->values);
    out->refs = c->refs;
    out->tables = c->tables;
    out->lens = c->lens;
    out->layers = c->layers;
    out->pages = (uint32_t)c->pages;
    out->sequences = (uint32_t)c->sequences;
    out->slots = (uint32_t)c->slots;
    out->heads = c->kv_heads;
    out->shift = __builtin_ctz((unsigned)c->page_size);
    out->dim = c->head_dim;
    out->bf16 = c->dtype == ACCEL_BF16;
    return ACCEL_OK;
}

// Entries of a list, at most: the kernels step over them by up to 1024 in 31 bits.
constexpr int64_t kMostEntries = INT32_MAX - 1024;

// A u32 vector of n entries (n < 0: any number); *len its length.
int check_list(const char* op, const char* what, const accel_tensor_t* t, int64_t n,
               int64_t* len) {
    char buf[256];
    if (!valid_tensor(t) || t->rank != 1 || t->dtype != ACCEL_U32 || t->shape[0] < 0) {
        snprintf(buf, sizeof buf, "%s must be a u32 vector", what);
        return refuse(op, buf);
    }
    if (t->shape[0] && !t->data) {
        snprintf(buf, sizeof buf, "%s is missing", what);
        return refuse(op, buf);
    }
    if (t->shape[0] > kMostEntries) {
        snprintf(buf, sizeof buf, "%s has %lld entries; up to %lld are served", what,
                 (long long)t->shape[0], (long long)kMostEntries);
        return refuse(op, buf);
    }
    if (n >= 0 && t->shape[0] != n) {
        snprintf(buf, sizeof buf, "%s has %lld entries and the call has %lld", what,
                 (long long)t->shape[0], (long long)n);
        return refuse(op, buf);
    }
    *len = t->shape[0];
    return ACCEL_OK;
}

// The sequences of a call of n entries (n < 0: as many as the list names): the
// list, or with NULL the cache's own order.
int check_seqs(const char* op, const accel_tensor_t* seqs, const KvCache& c, int64_t* n,
               const uint32_t** list) {
    char buf[256];
    *list = nullptr;
    if (!seqs) {
        if (*n < 0) *n = c.sequences;
        if (*n > (int64_t)c.sequences) {
            snprintf(buf, sizeof buf,
                     "%lld entries without a list of sequences, and the cache has %u",
                     (long long)*n, c.sequences);
            return refuse(op, buf);
        }
        return ACCEL_OK;
    }
    const int rc = check_list(op, "the list of sequences", seqs, *n, n);
    *list = static_cast<const uint32_t*>(seqs->data);
    return rc;
}

int check_layer(const char* op, const KvCache& c, int64_t layer) {
    char buf[128];
    if (layer >= 0 && layer < c.layers) return ACCEL_OK;
    snprintf(buf, sizeof buf, "layer %lld of a cache of %lld", (long long)layer,
             (long long)c.layers);
    return refuse(op, buf);
}

// Offsets of n entries over rows: u32 [n + 1].
int check_offsets(const char* op, const accel_tensor_t* t, int64_t* n) {
    int64_t len = 0;
    const int rc = check_list(op, "the offsets", t, -1, &len);
    if (rc != ACCEL_OK) return rc;
    if (len < 1) return refuse(op, "the offsets are one more than the entries and cannot be none");
    *n = len - 1;
    return ACCEL_OK;
}

bool same_rows(const accel_tensor_t* a, const accel_tensor_t* b) {
    return a->rank == b->rank && a->shape[0] == b->shape[0] && a->shape[1] == b->shape[1] &&
           a->shape[2] == b->shape[2];
}

// So many pieces of work an entry, below 2^31 in all, or a refusal.
int check_blocks(const char* op, int64_t n, int64_t each) {
    char buf[128];
    if (n <= INT32_MAX / each) return ACCEL_OK;
    snprintf(buf, sizeof buf, "%lld entries are more than a launch's 31-bit grid indexes",
             (long long)n);
    return refuse(op, buf);
}

// An open device with the submission counted, or a status.
int begin(int dev, Device** d) {
    *d = device(dev);
    return *d ? begin_submission(*d) : ACCEL_E_NO_DEVICE;
}

int done(Device* d, hipError_t e, int status, const char* what) {
    return status != ACCEL_OK ? status : classify(d, e, what);
}

}  // namespace

ACCEL_API int accel_kv_clear(int dev, void* stream, const accel_kv_cache_t* cache) {
    clear_error();
    KvCache c;
    int rc = check_cache("KVClear", cache, &c);
    if (rc != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK) return rc;
    return classify(d, launch_kv_clear((hipStream_t)stream, c), "KVClear launch");
}

ACCEL_API int accel_kv_reserve(int dev, void* stream, const accel_kv_cache_t* cache,
                               const accel_tensor_t* seqs, const accel_tensor_t* grow) {
    clear_error();
    const char* op = "KVReserve";
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    int64_t n = seqs ? -1 : (int64_t)c.sequences;
    if ((rc = check_list(op, "grow", grow, n, &n)) != ACCEL_OK) return rc;
    const uint32_t* list;
    if ((rc = check_seqs(op, seqs, c, &n, &list)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    int status = ACCEL_OK;
    const hipError_t e = launch_kv_reserve(d, (hipStream_t)stream, c, list,
                                           static_cast<const uint32_t*>(grow->data), (int)n,
                                           &status);
    return done(d, e, status, "KVReserve launch");
}

ACCEL_API int accel_kv_append(int dev, void* stream, const accel_kv_cache_t* cache,
                              int64_t layer, const accel_tensor_t* k, const accel_tensor_t* v,
                              const accel_tensor_t* seqs, const accel_tensor_t* offsets) {
    clear_error();
    const char* op = "KVAppend";
    char buf[256];
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    if ((rc = check_layer(op, c, layer)) != ACCEL_OK) return rc;
    if (!valid_tensor(k) || !valid_tensor(v)) return refuse(op, "an operand is missing");
    if (k->rank != 3 || !same_rows(k, v) || k->shape[0] < 0 || k->shape[1] != c.heads ||
        k->shape[2] != c.dim) {
        snprintf(buf, sizeof buf, "keys %s and values %s for a cache of %d heads of %d",
                 shape_str(k).c_str(), shape_str(v).c_str(), c.heads, c.dim);
        return refuse(op, buf);
    }
    if (k->dtype != v->dtype ||
        (k->dtype != ACCEL_F32 && k->dtype != ACCEL_F16 && k->dtype != ACCEL_BF16)) {
        snprintf(buf, sizeof buf, "keys are %s and values %s; both are f32, f16 or bf16",
                 dtype_name(k->dtype), dtype_name(v->dtype));
        return refuse(op, buf);
    }
    const int64_t T = k->shape[0];
    if (T > INT32_MAX / c.heads)
        return refuse(op, "more rows than a launch's 31-bit grid indexes");
    if (T && (!k->data || !v->data)) return refuse(op, "an operand is missing");
    if (!aligned16(k->data) || !aligned16(v->data))
        return refuse(op, "keys and values must start at 16-byte aligned addresses");
    int64_t n = T;
    const uint32_t *list, *off = nullptr;
    if (offsets) {
        if ((rc = check_offsets(op, offsets, &n)) != ACCEL_OK) return rc;
        off = static_cast<const uint32_t*>(offsets->data);
    }
    if ((rc = check_seqs(op, seqs, c, &n, &list)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0 || T == 0) return rc;
    return classify(d, launch_kv_append(d, (hipStream_t)stream, c, layer, k->data, v->data,
                                        k->dtype, list, off, (int)n, (int)T),
                    "KVAppend launch");
}

ACCEL_API int accel_kv_fork(int dev, void* stream, const accel_kv_cache_t* cache,
                            const accel_tensor_t* parents, const accel_tensor_t* children) {
    clear_error();
    const char* op = "KVFork";
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    int64_t n = -1;
    if ((rc = check_list(op, "the list of parents", parents, -1, &n)) != ACCEL_OK) return rc;
    if ((rc = check_list(op, "the list of children", children, n, &n)) != ACCEL_OK) return rc;
    if ((rc = check_blocks(op, n, 2 * c.layers + 1)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    int status = ACCEL_OK;
    const hipError_t e = launch_kv_fork(d, (hipStream_t)stream, c,
                                        static_cast<const uint32_t*>(parents->data),
                                        static_cast<const uint32_t*>(children->data), (int)n,
                                        &status);
    return done(d, e, status, "KVFork launch");
}

ACCEL_API int accel_kv_trim(int dev, void* stream, const accel_kv_cache_t* cache,
                            const accel_tensor_t* seqs, int64_t window, int64_t sinks) {
    clear_error();
    const char* op = "KVTrim";
    char buf[128];
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    if (window < 1 || sinks < 0) {
        snprintf(buf, sizeof buf, "a window of %lld with %lld sinks; it keeps one position or more",
                 (long long)window, (long long)sinks);
        return refuse(op, buf);
    }
    // no table holds as many positions; the kernel adds a page to the sinks
    if (window > INT32_MAX) window = INT32_MAX;
    if (sinks > INT32_MAX) sinks = INT32_MAX;
    int64_t n = -1;
    const uint32_t* list;
    if ((rc = check_seqs(op, seqs, c, &n, &list)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    return classify(d, launch_kv_free(d, (hipStream_t)stream, c, list, (int)n, window, sinks),
                    "KVTrim launch");
}

ACCEL_API int accel_kv_free(int dev, void* stream, const accel_kv_cache_t* cache,
                            const accel_tensor_t* seqs) {
    clear_error();
    const char* op = "KVFree";
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    int64_t n = -1;
    const uint32_t* list;
    if ((rc = check_seqs(op, seqs, c, &n, &list)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    return classify(d, launch_kv_free(d, (hipStream_t)stream, c, list, (int)n, 0, 0),
                    "KVFree launch");
}

ACCEL_API int accel_kv_compact(int dev, void* stream, const accel_kv_cache_t* cache,
                               accel_tensor_t* live) {
    clear_error();
    const char* op = "KVCompact";
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    int64_t one;
    if (live && (rc = check_list(op, "live", live, 1, &one)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK) return rc;
    int status = ACCEL_OK;
    const hipError_t e = launch_kv_compact(d, (hipStream_t)stream, c,
                                           live ? static_cast<uint32_t*>(live->data) : nullptr,
                                           &status);
    return done(d, e, status, "KVCompact launch");
}

ACCEL_API int accel_kv_copy(int dev, void* stream, const accel_kv_cache_t* cache,
                            const accel_tensor_t* src, const accel_tensor_t* dst) {
    clear_error();
    const char* op = "KVCopy";
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    int64_t n = -1;
    if ((rc = check_list(op, "the list of source pages", src, -1, &n)) != ACCEL_OK) return rc;
    if ((rc = check_list(op, "the list of target pages", dst, n, &n)) != ACCEL_OK) return rc;
    if ((rc = check_blocks(op, n, 2 * c.layers)) != ACCEL_OK) return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    return classify(d, launch_kv_copy(d, (hipStream_t)stream, c,
                                      static_cast<const uint32_t*>(src->data),
                                      static_cast<const uint32_t*>(dst->data), (int)n),
                    "KVCopy launch");
}

namespace {

int paged(const char* op, int dev, void* stream, const accel_tensor_t* q,
          const accel_tensor_t* offsets, bool ragged, const accel_kv_cache_t* cache,
          int64_t layer, const accel_tensor_t* seqs, const accel_attention_t* opt,
          accel_tensor_t* out, const accel_tensor_t* parents = nullptr, bool tree = false) {
    char buf[256];
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    if ((rc = check_layer(op, c, layer)) != ACCEL_OK) return rc;
    if (!valid_tensor(q)) return refuse(op, "the queries are missing");
    if (q->rank != 3 || q->shape[0] < 0 || q->shape[1] < 1 || q->shape[1] % c.heads ||
        q->shape[2] != c.dim) {
        snprintf(buf, sizeof buf,
                 "queries %s for a cache of %d heads of %d; they are [rows, heads, head_dim] "
                 "with heads a multiple of the cache's",
                 shape_str(q).c_str(), c.heads, c.dim);
        return refuse(op, buf);
    }
    const int32_t kv = c.bf16 ? ACCEL_BF16 : ACCEL_F16;
    if (q->dtype != ACCEL_F32 && q->dtype != kv) {
        snprintf(buf, sizeof buf, "queries are %s and the cache is %s; queries are f32 or the "
                 "cache's type", dtype_name(q->dtype), dtype_name(kv));
        return refuse(op, buf);
    }
    if (!valid_tensor(out) || out->dtype != q->dtype || out->rank != 3 || !same_rows(out, q))
        return refuse(op, "the output must have the queries' shape and type");
    const int64_t T = q->shape[0], H = q->shape[1];
    // a prompt's tiles of rows are at most two a row
    if (H > 65536 || T > INT32_MAX / 2 / H)
        return refuse(op, "more rows than a launch's 31-bit grid indexes");
    if (T && (!q->data || !out->data)) return refuse(op, "an operand is missing");
    if (!aligned16(q->data) || !aligned16(out->data))
        return refuse(op, "queries and output must start at 16-byte aligned addresses");
    Drafts a{};
    if (tree) {
        int64_t rows;
        if ((rc = check_list(op, "the list of parents", parents, T, &rows)) != ACCEL_OK) return rc;
        a.parents = static_cast<const uint32_t*>(parents->data);
    }
    if (opt) {
        // scores are in units of log 2: the scale times log2 e is finite too
        if (!(opt->scale >= 0 && opt->scale <= 0x1p127f) || opt->window < 0 || opt->sinks < 0) {
            snprintf(buf, sizeof buf,
                     "scale %g, window %lld and sinks %lld; none is negative and the scale is "
                     "finite, 2^127 at most",
                     (double)opt->scale, (long long)opt->window, (long long)opt->sinks);
            return refuse(op, buf);
        }
        a.scale = opt->scale;
        // past the positions a table can hold, a window is no window
        a.window = opt->window > INT32_MAX ? 0 : (uint32_t)opt->window;
        a.sinks = opt->sinks > INT32_MAX ? (uint32_t)INT32_MAX : (uint32_t)opt->sinks;
    }
    if (a.scale == 0) a.scale = (float)(1.0 / std::sqrt((double)c.dim));
    int64_t n = T;
    if (ragged) {
        if ((rc = check_offsets(op, offsets, &n)) != ACCEL_OK) return rc;
        a.offsets = static_cast<const uint32_t*>(offsets->data);
    }
    if ((rc = check_seqs(op, seqs, c, &n, &a.seqs)) != ACCEL_OK) return rc;
    a.n = (int)n;
    a.rows = (int)T;
    a.heads = (int)H;
    if (tree && !paged_tree_counts(c, a))
        return refuse(op, "more rows over such tables than 32 bits count the tiles of");
    if (!ragged && !paged_attention_counts(c, a))
        return refuse(op, "more entries of such tables than 32 bits count the tiles of");
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0 || T == 0) return rc;
    a.q = q->data;
    a.out = out->data;
    a.layer = layer;
    a.q_f32 = q->dtype == ACCEL_F32;
    int status = ACCEL_OK;
    const hipError_t e = tree     ? launch_paged_tree(d, (hipStream_t)stream, c, a, &status)
                         : ragged ? launch_paged_prefill(d, (hipStream_t)stream, c, a, &status)
                                  : launch_paged_attention(d, (hipStream_t)stream, c, a, &status);
    return done(d, e, status, op);
}

}  // namespace

ACCEL_API int accel_paged_attention(int dev, void* stream, const accel_tensor_t* q,
                                    const accel_kv_cache_t* cache, int64_t layer,
                                    const accel_tensor_t* seqs, const accel_attention_t* opt,
                                    accel_tensor_t* out) {
    clear_error();
    return paged("PagedAttention", dev, stream, q, nullptr, false, cache, layer, seqs, opt, out);
}

ACCEL_API int accel_paged_prefill(int dev, void* stream, const accel_tensor_t* q,
                                  const accel_tensor_t* offsets, const accel_kv_cache_t* cache,
                                  int64_t layer, const accel_tensor_t* seqs,
                                  const accel_attention_t* opt, accel_tensor_t* out) {
    clear_error();
    return paged("PagedPrefill", dev, stream, q, offsets, true, cache, layer, seqs, opt, out);
}

ACCEL_API int accel_paged_tree_attention(int dev, void* stream, const accel_tensor_t* q,
                                         const accel_tensor_t* offsets,
                                         const accel_tensor_t* parents,
                                         const accel_kv_cache_t* cache, int64_t layer,
                                         const accel_tensor_t* seqs,
                                         const accel_attention_t* opt, accel_tensor_t* out) {
    clear_error();
    return paged("PagedTreeAttention", dev, stream, q, offsets, true, cache, layer, seqs, opt, out,
                 parents, true);
}

namespace {

// A u32 matrix of one row an entry, up to 4096 wide.
int check_path(const char* op, const accel_tensor_t* t, int64_t n, int64_t* width) {
    char buf[256];
    if (!valid_tensor(t) || t->rank != 2 || t->dtype != ACCEL_U32 || t->shape[0] != n ||
        t->shape[1] < 1 || t->shape[1] > 4096) {
        snprintf(buf, sizeof buf,
                 "the paths must be u32 [%lld, width], a row an entry of 1 to 4096", (long long)n);
        return refuse(op, buf);
    }
    if (n && !t->data) return refuse(op, "the paths are missing");
    *width = t->shape[1];
    return check_blocks(op, n, *width);
}

}  // namespace

ACCEL_API int accel_tree_accept(int dev, void* stream, const accel_tensor_t* tokens,
                                const accel_tensor_t* parents, const accel_tensor_t* offsets,
                                const accel_tensor_t* sampled, accel_tensor_t* path,
                                accel_tensor_t* counts, accel_tensor_t* next) {
    clear_error();
    const char* op = "TreeAccept";
    int rc;
    int64_t T, n, len, width;
    if ((rc = check_list(op, "the list of tokens", tokens, -1, &T)) != ACCEL_OK ||
        (rc = check_list(op, "the list of parents", parents, T, &len)) != ACCEL_OK ||
        (rc = check_list(op, "the list of sampled tokens", sampled, T, &len)) != ACCEL_OK ||
        (rc = check_offsets(op, offsets, &n)) != ACCEL_OK ||
        (rc = check_path(op, path, n, &width)) != ACCEL_OK ||
        (rc = check_list(op, "the list of counts", counts, n, &len)) != ACCEL_OK ||
        (rc = check_list(op, "the list of next tokens", next, n, &len)) != ACCEL_OK)
        return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    const auto u32 = [](const accel_tensor_t* t) { return static_cast<uint32_t*>(t->data); };
    return classify(d, launch_tree_accept(d, (hipStream_t)stream, u32(tokens), u32(parents),
                                          u32(offsets), u32(sampled), T, n, width, u32(path),
                                          u32(counts), u32(next)),
                    "TreeAccept launch");
}

ACCEL_API int accel_kv_keep(int dev, void* stream, const accel_kv_cache_t* cache,
                            const accel_tensor_t* seqs, const accel_tensor_t* offsets,
                            const accel_tensor_t* path, const accel_tensor_t* counts) {
    clear_error();
    const char* op = "KVKeep";
    KvCache c;
    int rc = check_cache(op, cache, &c);
    if (rc != ACCEL_OK) return rc;
    int64_t n, len, width;
    const uint32_t* list;
    if ((rc = check_offsets(op, offsets, &n)) != ACCEL_OK ||
        (rc = check_path(op, path, n, &width)) != ACCEL_OK ||
        (rc = check_list(op, "the list of counts", counts, n, &len)) != ACCEL_OK ||
        (rc = check_seqs(op, seqs, c, &n, &list)) != ACCEL_OK)
        return rc;
    Device* d;
    if ((rc = begin(dev, &d)) != ACCEL_OK || n == 0) return rc;
    int status = ACCEL_OK;
    const hipError_t e = launch_kv_keep(d, (hipStream_t)stream, c, list,
                                        static_cast<const uint32_t*>(offsets->data),
                                        static_cast<const uint32_t*>(path->data), width,
                                        static_cast<const uint32_t*>(counts->data), n, &status);
    return done(d, e, status, "KVKeep launch");
}
