// kv_cache.cu -- the paged 8-bit key/value cache: appending a call's tokens,
// reading values back, and copying pages.  No counterpart in the reference
// (its generate loop keeps no keys or values, transformer.cu:986-1036).
//
// A value x of a (page, head) is held as the integer nearest to x / s, where s
// is the page's fp32 scale for that head.  Nearest means of the exact
// quotient: q = rint(x * (1/s)) is off by at most one, and the remainder
// x - q s, one FFMA, is exact wherever its size against s/2 matters (x and s
// have 24 bits, |q| <= 127, so a remainder of at most s is a whole number of
// ulps that fits 24 bits).  So the codes are a function of the inputs alone,
// not of the launch shape or of how a division is rounded.
#include "kv_cache.cuh"

namespace gbx {

constexpr float kTinyAmax = 7.888609052210118e-31f;   // 2^-100

// The integer nearest to x / s, ties to even; rs = 1/s rounded.  s > 0.
__device__ __forceinline__ int kv_code(float x, float s, float rs)
{
    float q = rintf(x * rs);
    const float r = fmaf(-q, s, x), h = 0.5f * s;
    if (fabsf(r) > h || (fabsf(r) == h && ((int)q & 1))) q += copysignf(1.0f, r);
    return (int)q;
}

// The page's scale for new values of largest size a; bad: one of them is not finite.
__device__ __forceinline__ float kv_new_scale(float a, bool bad)
{
    if (bad) return __int_as_float(0x7fc00000);
    return a >= kTinyAmax ? __fdiv_rn(a, 127.0f) : 0.0f;
}

// max of the two, NaN where either is
__device__ __forceinline__ float kv_max_scale(float a, float b) { return a != a || b != b ? a + b : fmaxf(a, b); }

// An earlier code under a larger scale: the integer nearest to c * old / now.
// The product has 31 bits and is exact in fp64, and the quotient of such
// numbers is never so near a half that its fp64 rounding could cross it.
__device__ __forceinline__ int kv_recode(int c, float old, float now)
{
    return (int)rint((double)c * (double)old / (double)now);
}

struct KvRows {
    const float* hi[2];   // K, V rows of the call
    const float* lo[2];
    int64_t ld;
};

// Where the call's block number j (0: the page of its first token) of a
// sequence lies: slots [s0, s0 + n), rows [i0, i0 + n) of the call.
struct KvBlock {
    int page_idx, s0, i0, n;
};

__device__ __forceinline__ KvBlock kv_block(const KvLayer& c, KvSeq q, int j)
{
    KvBlock k;
    const int first = q.len - q.n, P = 1 << c.log_page;
    k.page_idx = (first >> c.log_page) + j;
    const int p0 = k.page_idx << c.log_page;
    k.i0 = max(0, p0 - first);
    k.s0 = first + k.i0 - p0;
    k.n = min(P - k.s0, q.n - k.i0);
    return k;
}

// ---------------------------------------------------------------- append
// One warp per (sequence, block, K or V, head): the largest |x| of the
// block's new rows, the scale, the codes.  The rows are read twice, the
// second time from L1.
template <bool VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvLayer c, const KvRows r, int64_t units, int blocks)
{
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (u >= units) return;
    const int h = (int)(u % c.heads);
    int64_t w = u / c.heads;
    const int which = (int)(w & 1);
    w >>= 1;
    const int j = (int)(w % blocks), b = (int)(w / blocks);
    bool bad_len;
    const KvSeq q = kv_seq(c, b, &bad_len);
    if (bad_len && lane == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    const KvBlock k = kv_block(c, q, j);
    if (k.n <= 0) return;
    const int page = kv_page(c, b, k.page_idx);
    if (page < 0) {
        if (lane == 0) kv_flag(c.err, GBX_KV_BAD_PAGE);
        return;
    }
    const int hd = c.hd, P = 1 << c.log_page;
    const float* hi = r.hi[which] + ((int64_t)b * c.S + k.i0) * r.ld + (int64_t)h * hd;
    const float* lo = r.lo[which] ? r.lo[which] + (hi - r.hi[which]) : nullptr;
    const int64_t ph = (int64_t)page * c.heads + h;
    int8_t* codes = (which ? c.v : c.k) + ph * P * hd;
    float* scale = (which ? c.vs : c.ks) + ph;
    const int quads = hd >> 2, n4 = k.n * quads;   // groups of 4 values
    auto load = [&](int e) -> float4 {
        const int64_t at = (int64_t)(e / quads) * r.ld + (e % quads) * 4;
        float4 x;
        if (VEC) {
            x = *reinterpret_cast<const float4*>(hi + at);
            if (lo) x = add4(x, *reinterpret_cast<const float4*>(lo + at));
        } else {
            x = make_float4(hi[at], hi[at + 1], hi[at + 2], hi[at + 3]);
            if (lo) x = add4(x, make_float4(lo[at], lo[at + 1], lo[at + 2], lo[at + 3]));
        }
        return x;
    };
    float a = 0.0f;
    bool bad = false;
    for (int e = lane; e < n4; e += 32) {
        const float4 x = load(e);
        const float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        bad |= !(x.x - x.x == 0.0f) | !(x.y - x.y == 0.0f) | !(x.z - x.z == 0.0f) | !(x.w - x.w == 0.0f);
        a = fmaxf(a, m);
    }
    a = group_max<32>(a);
    bad = __any_sync(0xffffffffu, bad);
    float s = kv_new_scale(a, bad);
    if (k.s0 > 0) {
        const float old = *scale;
        s = kv_max_scale(old, s);
        if (s != old) {   // grew, or turned NaN: the earlier slots' codes
            for (int e = lane; e < k.s0 * hd; e += 32) {
                const int t = e / hd, i = e % hd;
                int8_t* p = codes + (which ? ((t >> 4) * hd + i) * 16 + (t & 15) : t * hd + i);
                *p = (int8_t)(s > 0.0f ? kv_recode(*p, old, s) : 0);
            }
        }
    }
    __syncwarp();
    if (lane == 0) *scale = s;
    const bool live = s > 0.0f;   // false for 0 and NaN: codes 0
    const float rs = 1.0f / s;
    for (int e = lane; e < n4; e += 32) {
        const float4 x = load(e);
        const int t = k.s0 + e / quads, i = (e % quads) * 4;
        char4 q4 = make_char4(0, 0, 0, 0);
        if (live) {
            q4.x = (signed char)kv_code(x.x, s, rs);
            q4.y = (signed char)kv_code(x.y, s, rs);
            q4.z = (signed char)kv_code(x.z, s, rs);
            q4.w = (signed char)kv_code(x.w, s, rs);
        }
        if (which) {
            int8_t* p = codes + ((t >> 4) * hd + i) * 16 + (t & 15);
            p[0] = q4.x;
            p[16] = q4.y;
            p[32] = q4.z;
            p[48] = q4.w;
        } else {
            *reinterpret_cast<char4*>(codes + t * hd + i) = q4;
        }
    }
}

// ---------------------------------------------------------------- read back
// One thread per four values of a row.
template <bool VEC>
__global__ void __launch_bounds__(256)
kv_read_kernel(const KvLayer c, float* k_out, float* v_out, int64_t ld, int64_t units)
{
    grid_dependency_wait();
    const int quads = c.hd >> 2, row4 = c.heads * quads;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.x * 256) {
        const int64_t row = u / row4;
        const int x = (int)(u - row * row4), h = x / quads, i = (x - h * quads) * 4;
        const int b = (int)(row / c.S), ri = (int)(row - (int64_t)b * c.S);
        bool bad_len;
        const KvSeq q = kv_seq(c, b, &bad_len);
        if (bad_len && ri == 0 && x == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
        if (ri >= q.n) continue;
        const int t = q.len - q.n + ri, P = 1 << c.log_page, slot = t & (P - 1);
        const int page = kv_page(c, b, t >> c.log_page);
        if (page < 0) {
            if (x == 0) kv_flag(c.err, GBX_KV_BAD_PAGE);
            continue;
        }
        const int64_t ph = (int64_t)page * c.heads + h;
        for (int which = 0; which < 2; ++which) {
            float* out = which ? v_out : k_out;
            if (!out) continue;
            const float s = (which ? c.vs : c.ks)[ph];
            const int8_t* p = (which ? c.v : c.k) + ph * P * c.hd;
            char4 q4;
            if (which) {
                p += ((slot >> 4) * c.hd + i) * 16 + (slot & 15);
                q4 = make_char4(p[0], p[16], p[32], p[48]);
            } else {
                q4 = *reinterpret_cast<const char4*>(p + slot * c.hd + i);
            }
            const float4 f = make_float4(q4.x * s, q4.y * s, q4.z * s, q4.w * s);
            float* o = out + row * ld + (int64_t)h * c.hd + i;
            if (VEC) {
                *reinterpret_cast<float4*>(o) = f;
            } else {
                o[0] = f.x;
                o[1] = f.y;
                o[2] = f.z;
                o[3] = f.w;
            }
        }
    }
}

// ---------------------------------------------------------------- page copies
struct KvPool {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    int64_t page_bytes;    // heads * page * hd, a multiple of 256
    int64_t pages;
    int heads, layers;
    int32_t* err;
};

// One CTA per (pair, layer, K or V).  A page of a layer is one contiguous
// run of bytes.  Before it stores, the CTA looks its target up among all
// sources and earlier targets (n words each, from L2): a pair that would race
// with another is left out, by every CTA alike.
__global__ void __launch_bounds__(256)
kv_copy_kernel(const KvPool c, const int32_t* src, const int32_t* dst, int n)
{
    grid_dependency_wait();
    const int i = blockIdx.x, layer = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int from = src[i], to = dst[i];
    const bool first = blockIdx.y == 0 && threadIdx.x == 0;
    if ((uint64_t)(int64_t)from >= (uint64_t)c.pages || (uint64_t)(int64_t)to >= (uint64_t)c.pages) {
        if (first) kv_flag(c.err, GBX_KV_BAD_PAGE);
        return;
    }
    if (from == to) return;
    bool clash = false;
    for (int j = threadIdx.x; j < n; j += 256) clash |= (src[j] == to) | (j < i && dst[j] == to);
    if (__syncthreads_or(clash)) {
        if (first) kv_flag(c.err, GBX_KV_BAD_PAIR);
        return;
    }
    int8_t* base = (which ? c.v : c.k) + (int64_t)layer * c.pages * c.page_bytes;
    const uint4* s = reinterpret_cast<const uint4*>(base + from * c.page_bytes);
    uint4* d = reinterpret_cast<uint4*>(base + to * c.page_bytes);
    for (int64_t e = threadIdx.x; e < c.page_bytes >> 4; e += 256) d[e] = s[e];
    float* sc = (which ? c.vs : c.ks) + (int64_t)layer * c.pages * c.heads;
    for (int e = threadIdx.x; e < c.heads; e += 256) sc[(int64_t)to * c.heads + e] = sc[(int64_t)from * c.heads + e];
}

// ---------------------------------------------------------------- host checks
int kv_check_cache(const gbx_kv_cache* c, const char* what)
{
    if (!c) return set_error(GBX_EINVAL, "%s: null cache", what);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return set_error(GBX_EINVAL, "%s: the cache has a null array", what);
    if (c->layers <= 0 || c->heads <= 0 || c->pages <= 0)
        return set_error(GBX_EINVAL, "%s: cache of %d layers, %lld pages, %d heads", what, c->layers,
                         (long long)c->pages, c->heads);
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return set_error(GBX_EINVAL, "%s: %d tokens per page (16, 32, 64 or 128)", what, c->page);
    if (c->hd < 16 || c->hd > 128 || c->hd % 16)
        return set_error(GBX_EINVAL, "%s: head width %d (a multiple of 16 up to 128)", what, c->hd);
    if (c->pages > 0x7fffffffLL || c->heads > 65536 || c->layers > 32767)
        return set_error(GBX_ERANGE, "%s: cache too large", what);
    if (!aligned16(c->k) || !aligned16(c->v) || ((uintptr_t)c->k_scale & 3) || ((uintptr_t)c->v_scale & 3))
        return set_error(GBX_EINVAL, "%s: the cache's code arrays need 16-byte alignment, its scales 4", what);
    return GBX_OK;
}

int kv_layer(const gbx_kv_cache* c, int layer, const int32_t* table, int max_pages, const int32_t* kv_len,
             const int32_t* n_new, int B, int S, int* err, const char* what, KvLayer* out)
{
    if (int rc = kv_check_cache(c, what)) return rc;
    if (layer < 0 || layer >= c->layers)
        return set_error(GBX_EINVAL, "%s: layer %d of %d", what, layer, c->layers);
    if (B < 0 || S < 0 || max_pages < 0)
        return set_error(GBX_EINVAL, "%s: B=%d S=%d max_pages=%d", what, B, S, max_pages);
    if ((int64_t)max_pages * c->page > (1 << 30))   // token indexes, and sums of two of them, are ints
        return set_error(GBX_ERANGE, "%s: %d pages of %d tokens", what, max_pages, c->page);
    if ((int64_t)B * S > 0x7fffffffLL) return set_error(GBX_ERANGE, "%s: B=%d S=%d", what, B, S);
    if (B > 0 && S > 0 && (!table || !kv_len || max_pages == 0))
        return set_error(GBX_EINVAL, "%s: null or empty table, or null kv_len", what);
    int lg = 4;
    while ((1 << lg) < c->page) ++lg;
    const int64_t codes = (int64_t)layer * c->pages * c->heads * c->page * c->hd;
    const int64_t scales = (int64_t)layer * c->pages * c->heads;
    out->k = c->k + codes;
    out->v = c->v + codes;
    out->ks = c->k_scale + scales;
    out->vs = c->v_scale + scales;
    out->table = table;
    out->kv_len = kv_len;
    out->n_new = n_new;
    out->pages = (int32_t)c->pages;
    out->max_pages = max_pages;
    out->heads = c->heads;
    out->hd = c->hd;
    out->log_page = lg;
    out->S = S;
    out->err = err;
    return GBX_OK;
}

}  // namespace gbx

using namespace gbx;

extern "C" int gbx_kv_append(const gbx_kv_cache* cache_host, int layer, const int32_t* table, int max_pages,
                             const int32_t* kv_len, const int32_t* n_new, int B, int S, const float* k_hi,
                             const float* k_lo, const float* v_hi, const float* v_lo, int64_t ld, int* err_flag,
                             gbx_stream_t stream)
{
    KvLayer c;
    if (int rc = kv_layer(cache_host, layer, table, max_pages, kv_len, n_new, B, S, err_flag, "gbx_kv_append", &c))
        return rc;
    if (B == 0 || S == 0) return GBX_OK;
    if (!k_hi || !v_hi) return set_error(GBX_EINVAL, "gbx_kv_append: null pointer");
    if (ld < (int64_t)c.heads * c.hd)
        return set_error(GBX_EINVAL, "gbx_kv_append: ld=%lld < heads*hd", (long long)ld);
    // blocks a sequence's S tokens can touch
    const int P = 1 << c.log_page;
    const int64_t touched = ((int64_t)S + 2 * P - 2) / P;
    const int blocks = (int)(touched < max_pages ? touched : max_pages);
    const int64_t units = (int64_t)B * blocks * 2 * c.heads;
    if ((units + 7) / 8 > 0x7fffffffLL) return set_error(GBX_ERANGE, "gbx_kv_append: B=%d S=%d heads=%d", B, S, c.heads);
    KvRows r;
    r.hi[0] = k_hi;
    r.hi[1] = v_hi;
    r.lo[0] = k_lo;
    r.lo[1] = v_lo;
    r.ld = ld;
    const bool vec = aligned16(k_hi) && aligned16(v_hi) && aligned16(k_lo) && aligned16(v_lo) && ld % 4 == 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((units + 7) / 8));
    if (vec) launch_row_kernel(kv_append_kernel<true>, grid, dim3(256), 0, s, c, r, units, blocks);
    else launch_row_kernel(kv_append_kernel<false>, grid, dim3(256), 0, s, c, r, units, blocks);
    return check_launch("gbx_kv_append");
}

extern "C" int gbx_kv_read(const gbx_kv_cache* cache_host, int layer, const int32_t* table, int max_pages,
                           const int32_t* kv_len, const int32_t* n, int B, int S, float* k_out, float* v_out,
                           int64_t ld, int* err_flag, gbx_stream_t stream)
{
    KvLayer c;
    if (int rc = kv_layer(cache_host, layer, table, max_pages, kv_len, n, B, S, err_flag, "gbx_kv_read", &c)) return rc;
    if (B == 0 || S == 0 || (!k_out && !v_out)) return GBX_OK;
    if (ld < (int64_t)c.heads * c.hd) return set_error(GBX_EINVAL, "gbx_kv_read: ld=%lld < heads*hd", (long long)ld);
    const int64_t units = (int64_t)B * S * c.heads * (c.hd / 4);
    const bool vec = aligned16(k_out) && aligned16(v_out) && ld % 4 == 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int grid = vec ? persistent_grid(kv_read_kernel<true>, 256, 0, (units + 255) / 256, 8)
                         : persistent_grid(kv_read_kernel<false>, 256, 0, (units + 255) / 256, 8);
    if (grid < 0) return GBX_ECUDA;
    if (vec) launch_row_kernel(kv_read_kernel<true>, dim3(grid), dim3(256), 0, s, c, k_out, v_out, ld, units);
    else launch_row_kernel(kv_read_kernel<false>, dim3(grid), dim3(256), 0, s, c, k_out, v_out, ld, units);
    return check_launch("gbx_kv_read");
}

extern "C" int gbx_kv_copy_pages(const gbx_kv_cache* cache_host, const int32_t* src, const int32_t* dst, int n,
                                 int* err_flag, gbx_stream_t stream)
{
    if (int rc = kv_check_cache(cache_host, "gbx_kv_copy_pages")) return rc;
    if (n < 0) return set_error(GBX_EINVAL, "gbx_kv_copy_pages: n=%d", n);
    if (n == 0) return GBX_OK;
    if (!src || !dst) return set_error(GBX_EINVAL, "gbx_kv_copy_pages: null pointer");
    const gbx_kv_cache& h = *cache_host;
    KvPool c;
    c.k = h.k;
    c.v = h.v;
    c.ks = h.k_scale;
    c.vs = h.v_scale;
    c.page_bytes = (int64_t)h.heads * h.page * h.hd;
    c.pages = h.pages;
    c.heads = h.heads;
    c.layers = h.layers;
    c.err = err_flag;
    launch_row_kernel(kv_copy_kernel, dim3((unsigned)n, (unsigned)h.layers * 2), dim3(256), 0,
                      reinterpret_cast<cudaStream_t>(stream), c, src, dst, n);
    return check_launch("gbx_kv_copy_pages");
}
