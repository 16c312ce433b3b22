// kv_cache.cuh -- one layer of the paged 8-bit key/value cache as the kernels
// see it, and the checks its entry points share.
#pragma once

#include "gbx_common.cuh"

namespace gbx {

// One layer.  `page` is a power of two >= 16: token t of a page's slot
// s = t & (page - 1) lies in its 16-token group s >> 4.
struct KvLayer {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    const int32_t* table;
    const int32_t* kv_len;
    const int32_t* n_new;   // NULL: S for every sequence
    int32_t pages, max_pages, heads, hd, log_page, S;
    int32_t* err;
};

// Plain loads throughout: an earlier kernel on the stream may have written any
// of these arrays, and a read-only (ld.nc) load could be moved above the wait
// for it.
//
// The sequence's rows: n of them, the last at token len - 1.  A sequence whose
// numbers are out of range counts as one with no rows and no tokens.
struct KvSeq {
    int len, n;
};

__device__ __forceinline__ KvSeq kv_seq(const KvLayer& c, int b, bool* bad)
{
    KvSeq s;
    s.len = c.kv_len[b];
    s.n = c.n_new ? c.n_new[b] : c.S;
    *bad = s.n < 0 || s.n > c.S || s.len < s.n || (int64_t)s.len > ((int64_t)c.max_pages << c.log_page);
    if (*bad) s.len = s.n = 0;
    return s;
}

// Page of the sequence's j-th block, or -1 for one outside the pool.
__device__ __forceinline__ int kv_page(const KvLayer& c, int b, int j)
{
    const int p = c.table[(int64_t)b * c.max_pages + j];
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}

__device__ __forceinline__ void kv_flag(int32_t* err, int bit)
{
    if (err) atomicOr(err, bit);
}

// Host checks shared by the entry points that address a layer through a table.
int kv_check_cache(const gbx_kv_cache* c, const char* what);
int kv_layer(const gbx_kv_cache* c, int layer, const int32_t* table, int max_pages, const int32_t* kv_len,
             const int32_t* n_new, int B, int S, int* err, const char* what, KvLayer* out);

// Page src[i] of one pool becomes page dst[i] of another of the same layers, heads,
// page and hd (or of the same pool, as gbx_kv_copy_pages), in every layer.
int kv_copy_across(const gbx_kv_cache* from, const gbx_kv_cache* to, const int32_t* src, const int32_t* dst, int n, int* err,
                   gbx_stream_t stream);

}  // namespace gbx
