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

// Four values' codes at scale s > 0 (rs = 1/s rounded), one to a byte: the
// integers nearest to x / s, ties to even.  Adding 1.5 2^23 rounds x rs and
// leaves the integer in the low mantissa bits.  Where a remainder reaches s/2
// (a tie, or a neighbour of one: about one value in 10^5) the integer is
// settled by it.
constexpr float kKvMagic = 12582912.0f;

__device__ __forceinline__ uint32_t kv_codes4(float4 x, float s, float rs)
{
    const float2 magic = splat2(kKvMagic), by = splat2(rs), neg = splat2(-s);
    float2 a = __ffma2_rn(lo2(x), by, magic), b = __ffma2_rn(hi2(x), by, magic);
    const float2 qa = __fadd2_rn(a, splat2(-kKvMagic)), qb = __fadd2_rn(b, splat2(-kKvMagic));
    const float2 ra = __ffma2_rn(qa, neg, lo2(x)), rb = __ffma2_rn(qb, neg, hi2(x));
    const float h = 0.5f * s;
    if (fmaxf(fmaxf(fabsf(ra.x), fabsf(ra.y)), fmaxf(fabsf(rb.x), fabsf(rb.y))) >= h) {
        auto settle = [&](float& m, float q, float r) {
            if (fabsf(r) > h || (fabsf(r) == h && ((int)q & 1))) m += copysignf(1.0f, r);
        };
        settle(a.x, qa.x, ra.x);
        settle(a.y, qa.y, ra.y);
        settle(b.x, qb.x, rb.x);
        settle(b.y, qb.y, rb.y);
    }
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                       __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

// The page's scale for new values of largest size a; bad: one of them is not finite.
__device__ __forceinline__ float kv_new_scale(float a, bool bad)
{
    if (bad) return __int_as_float(0x7fc00000);
    return a >= kTinyAmax ? __fdiv_rn(a, 127.0f) : 0.0f;
}

// max of the two, NaN where either is
__device__ __forceinline__ float kv_max_scale(float a, float b) { return a != a || b != b ? a + b : fmaxf(a, b); }

// Sixteen earlier codes under a larger scale, the first n of them: the integers
// nearest to c * old / now, ties to even.  ratio is old / now rounded to fp64, so
// c * ratio is off by less than 2^-44.  A quotient that is no tie keeps 2^-34 from one:
// near a tie |c| old / now is about a half or more, so now's exponent is at most 9
// above old's, and 2 c old - (odd) now is at least one unit of their 24 bits.  A tie
// itself shows in the remainder, which is exact: c * old and q * now have 31 bits.
__device__ __forceinline__ uint4 kv_recode16(uint4 w, int n, double old, double now, double ratio)
{
    uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const double c = (double)(int8_t)(x[e >> 2] >> (8 * (e & 3)));
        double q = rint(c * ratio);
        const double rem = fma(-q, now, c * old), h = 0.5 * now;
        if (fabs(rem) > h || (fabs(rem) == h && ((int)q & 1))) q += copysign(1.0, rem);
        const uint32_t code = now > 0.0 ? (uint32_t)(int)q & 255u : 0u;
        if (e < n) x[e >> 2] = (x[e >> 2] & ~(255u << (8 * (e & 3)))) | code << (8 * (e & 3));
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
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
constexpr int kKvHeld = 4;   // groups of four values a lane holds between the maximum and the codes

struct KvAppend {
    KvLayer c;
    KvRows r;
    FastDiv by_quads, by_heads, by_blocks;   // unit = ((b * blocks + j) * 2 + which) * heads + h
    int blocks;
    uint32_t units;
};

struct KvUnit {
    int h, which, j, b;
};

__device__ __forceinline__ KvUnit kv_unit(uint32_t u, int heads, FastDiv by_heads, int blocks, FastDiv by_blocks)
{
    KvUnit k;
    const uint32_t w = fast_div(u, by_heads), v = w >> 1;
    k.h = (int)(u - w * heads);
    k.which = (int)(w & 1);
    k.b = (int)fast_div(v, by_blocks);
    k.j = (int)(v - k.b * blocks);
    return k;
}

__device__ __forceinline__ float kv_abs4(float4 x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); }

// 0, or NaN where an entry is not finite
__device__ __forceinline__ float kv_bad4(float4 x) { return fmaf(x.x, 0.0f, fmaf(x.y, 0.0f, fmaf(x.z, 0.0f, x.w * 0.0f))); }

template <bool VEC>
__device__ __forceinline__ float4 kv_load4(const float* hi, const float* lo, int64_t at)
{
    float4 x;
    if (VEC) {
        x = *reinterpret_cast<const float4*>(hi + at);
        if (lo) x = add4(x, *reinterpret_cast<const float4*>(lo + at));
    } else {
        x = make_float4(hi[at], hi[at + 1], hi[at + 2], hi[at + 3]);
        if (lo) x = add4(x, make_float4(lo[at], lo[at + 1], lo[at + 2], lo[at + 3]));
    }
    return x;
}

// The page's scale (old, where it holds earlier slots) with new values of largest
// size amax in, and where it grew the codes before slot s0 recoded by `threads`
// threads, this one the id-th.  Called by all of them, which have to meet before
// *scale is stored.  By words of 16 codes: one by one, a warp waited for memory some 80
// times in a page of 40 tokens (32 sequences x 12 heads of width 64: 43 us a growing step, now 12).
__device__ __forceinline__ float kv_grow(const KvBlock& k, int8_t* codes, float old, float amax, bool bad, int which, int hd,
                                         int id, int threads)
{
    float s = kv_new_scale(amax, bad);
    if (k.s0 > 0) {
        s = kv_max_scale(old, s);
        if (s != old) {   // grew, or turned NaN
            // words of 16 codes: of one token, or of one column and 16 tokens, the last of which may be new slots'
            const double ratio = (double)old / (double)s;
            const int words = which ? ((k.s0 + 15) >> 4) * hd : k.s0 * hd >> 4;
            for (int e = id; e < words; e += threads) {
                uint4* p = reinterpret_cast<uint4*>(codes) + e;
                *p = kv_recode16(*p, which ? k.s0 - 16 * (e / hd) : 16, (double)old, (double)s, ratio);
            }
        }
    }
    return s;
}

// Few new rows per sequence (a decode step, drafts): one warp per (sequence, block, K or V, head), the
// largest |x| of the block's new rows, the scale, the codes.  The first 512
// values are held in registers, others read again from L1.  Latency bounds it
// (length, rows and page, scale, codes one after another): 2.9 us for 32 sequences x
// 12 heads, 8.6 for 256 x 25.
template <bool VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppend a)
{
    grid_dependency_wait();
    const KvLayer& c = a.c;
    const int lane = threadIdx.x & 31;
    const uint32_t unit = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= a.units) return;
    const KvUnit u = kv_unit(unit, c.heads, a.by_heads, a.blocks, a.by_blocks);
    bool bad_len;
    const KvSeq q = kv_seq(c, u.b, &bad_len);
    if (bad_len && lane == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    const KvBlock k = kv_block(c, q, u.j);
    if (k.n <= 0) return;
    const int page = kv_page(c, u.b, k.page_idx);   // not waited for before the rows are asked for
    const int hd = c.hd;
    const float* base = a.r.hi[u.which];
    const float* hi = base + ((int64_t)u.b * c.S + k.i0) * a.r.ld + (int64_t)u.h * hd;
    const float* lo = a.r.lo[u.which] ? a.r.lo[u.which] + (hi - base) : nullptr;
    const int quads = hd >> 2, n4 = k.n * quads;   // groups of 4 values
    auto load = [&](int e) {
        const int r = (int)fast_div(e, a.by_quads);
        return kv_load4<VEC>(hi, lo, r * a.r.ld + (e - r * quads) * 4);
    };
    float4 held[kKvHeld];
#pragma unroll
    for (int i = 0; i < kKvHeld; ++i) held[i] = lane + 32 * i < n4 ? load(lane + 32 * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (page < 0) {
        if (lane == 0) kv_flag(c.err, GBX_KV_BAD_PAGE);
        return;
    }
    const int64_t ph = (int64_t)page * c.heads + u.h;
    int8_t* codes = (u.which ? c.v : c.k) + (ph << c.log_page) * hd;
    float* scale = (u.which ? c.vs : c.ks) + ph;
    float amax = 0.0f, bad = 0.0f;
    auto look = [&](float4 x) {
        amax = fmaxf(amax, kv_abs4(x));
        bad += kv_bad4(x);
    };
    const float old = k.s0 > 0 ? *scale : 0.0f;    // asked for before the maximum is formed
#pragma unroll
    for (int i = 0; i < kKvHeld; ++i) look(held[i]);
    for (int e = lane + 32 * kKvHeld; e < n4; e += 32) look(load(e));
    amax = group_max<32>(amax);
    const float s = kv_grow(k, codes, old, amax, __any_sync(0xffffffffu, bad != bad), u.which, hd, lane, 32);
    __syncwarp();
    if (lane == 0) *scale = s;
    const bool live = s > 0.0f;   // false for 0 and NaN: codes 0
    const float rs = 1.0f / s;
    auto put = [&](int e, float4 x) {
        const int r = (int)fast_div(e, a.by_quads), i = (e - r * quads) * 4, t = k.s0 + r;
        const uint32_t q4 = live ? kv_codes4(x, s, rs) : 0u;
        if (u.which) {
            int8_t* p = codes + ((t >> 4) * hd + i) * 16 + (t & 15);
#pragma unroll
            for (int m = 0; m < 4; ++m) p[16 * m] = (int8_t)(q4 >> (8 * m));
        } else {
            *reinterpret_cast<uint32_t*>(codes + t * hd + i) = q4;
        }
    };
#pragma unroll
    for (int i = 0; i < kKvHeld; ++i)
        if (lane + 32 * i < n4) put(lane + 32 * i, held[i]);
    for (int e = lane + 32 * kKvHeld; e < n4; e += 32) put(e, load(e));
}

// Many new rows: one CTA per (sequence, block, K or V, head), a warp for every
// 16 slots x 64 columns, 32 values to a lane held in registers between the
// maximum and the codes, so each row is read once.  Keys: a lane has four
// columns of every other slot (16-byte loads, 4-byte stores, a row's in
// line); values: two columns of all 16 slots, whose codes are two 16-byte words
// of the 16-tokens-innermost layout.  HBM bounds it: 32.8 us for 8 prompts of 1024
// rows of 25 heads x 64 (131 MB, 4.0 TB/s), the rest the CTAs' start.
template <bool VEC>
__global__ void __launch_bounds__(512) kv_append_pages_kernel(const KvAppend a)
{
    grid_dependency_wait();
    __shared__ float s_max[16], s_bad[16];
    const KvLayer& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const KvUnit u = kv_unit(blockIdx.x, c.heads, a.by_heads, a.blocks, a.by_blocks);
    bool bad_len;
    const KvSeq q = kv_seq(c, u.b, &bad_len);
    if (bad_len && threadIdx.x == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    const KvBlock k = kv_block(c, q, u.j);
    if (k.n <= 0) return;
    const int hd = c.hd;
    const int page = kv_page(c, u.b, k.page_idx);   // not waited for before the rows are asked for
    // this warp's slots t0 .. t0 + 15 and columns c0 .. c0 + 63
    const int halves = hd > 64 ? 2 : 1;
    const int t0 = 16 * (halves == 2 ? warp >> 1 : warp), c0 = halves == 2 ? 64 * (warp & 1) : 0;
    const float* base = a.r.hi[u.which];
    // row of slot 0 (which may lie before the call's rows)
    const float* hi = base + ((int64_t)u.b * c.S + k.i0 - k.s0) * a.r.ld + (int64_t)u.h * hd;
    const float* lo = a.r.lo[u.which] ? a.r.lo[u.which] + (hi - base) : nullptr;
    const int ks0 = k.s0, ks1 = k.s0 + k.n;   // the slots to be filled
    // values: x[i] = slots 2i, 2i + 1 x two columns.  All of a plane's loads are
    // issued before any is used.
    const int col = u.which ? c0 + 2 * lane : c0 + 4 * (lane & 15);
    const bool in = col < hd;
    auto plane = [&](const float* src, float4 (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (u.which == 0) {
                const int t = t0 + 2 * i + (lane >> 4);
                const float* at = src + t * a.r.ld + col;
                if (in && t >= ks0 && t < ks1) x[i] = VEC ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
            } else {
                const int t = t0 + 2 * i;
                const float* at = src + t * a.r.ld + col;
                float2 y = make_float2(0.0f, 0.0f), z = y;
                if (in && t >= ks0 && t < ks1) y = VEC ? *reinterpret_cast<const float2*>(at) : make_float2(at[0], at[1]);
                at += a.r.ld;
                if (in && t + 1 >= ks0 && t + 1 < ks1) z = VEC ? *reinterpret_cast<const float2*>(at) : make_float2(at[0], at[1]);
                x[i] = cat2(y, z);
            }
        }
    };
    float4 x[8];
    plane(hi, x);
    if (lo) {
        float4 y[8];
        plane(lo, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = add4(x[i], y[i]);
    }
    float amax = 0.0f, bad = 0.0f;
    if (page < 0) {   // the CTA's threads alike
        if (threadIdx.x == 0) kv_flag(c.err, GBX_KV_BAD_PAGE);
        return;
    }
    const int64_t ph = (int64_t)page * c.heads + u.h;
    int8_t* codes = (u.which ? c.v : c.k) + (ph << c.log_page) * hd;
    float* scale = (u.which ? c.vs : c.ks) + ph;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, kv_abs4(x[i]));
        bad += kv_bad4(x[i]);
    }
    amax = group_max<32>(amax);
    bad = group_sum<32>(bad);
    if (lane == 0) {
        s_max[warp] = amax;
        s_bad[warp] = bad;
    }
    __syncthreads();
    for (int w = 0; w < warps; ++w) {
        amax = fmaxf(amax, s_max[w]);
        bad += s_bad[w];
    }
    const float s = kv_grow(k, codes, k.s0 > 0 ? *scale : 0.0f, amax, bad != bad, u.which, hd, threadIdx.x, blockDim.x);
    __syncthreads();   // every thread has read the old scale, and recoded what it recodes
    if (threadIdx.x == 0) *scale = s;
    if (col >= hd) return;
    const bool live = s > 0.0f;
    const float rs = 1.0f / s;
    uint32_t q4[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        q4[i] = live ? kv_codes4(x[i], s, rs) : 0u;
    if (u.which == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = t0 + 2 * i + (lane >> 4);
            if (t >= ks0 && t < ks1) *reinterpret_cast<uint32_t*>(codes + t * hd + col) = q4[i];
        }
    } else {
        // q4[i]: bytes (slot 2i: columns 0, 1; slot 2i + 1: columns 0, 1)
        int8_t* to = codes + ((t0 >> 4) * hd + col) * 16;
        uint32_t w[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[0][i] = __byte_perm(q4[2 * i], q4[2 * i + 1], 0x6420);
            w[1][i] = __byte_perm(q4[2 * i], q4[2 * i + 1], 0x7531);
        }
        if (ks0 <= t0 && t0 + 16 <= ks1) {
            *reinterpret_cast<uint4*>(to) = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
            *reinterpret_cast<uint4*>(to + 16) = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
        } else {
#pragma unroll
            for (int t = 0; t < 16; ++t)
                if (t0 + t >= ks0 && t0 + t < ks1) {
                    to[t] = (int8_t)(w[0][t >> 2] >> (8 * (t & 3)));
                    to[16 + t] = (int8_t)(w[1][t >> 2] >> (8 * (t & 3)));
                }
        }
    }
}

// ---------------------------------------------------------------- read back
// One warp per (sequence, 16-token group, K or V, head).  Keys: a lane takes four
// columns of a token; values: one column of all 16 tokens, a 16-byte load, and
// stores row by row, 32 columns in line.  HBM bounds it: 5.1 TB/s for 8 x 1087 rows
// of 25 heads x 64; five CTAs to an SM (8 with spills 4.1, 3 by registers 2.7).
template <bool VEC>
__global__ void __launch_bounds__(256, 5)
kv_read_kernel(const KvLayer c, float* k_out, float* v_out, int64_t ld, FastDiv by_heads, int groups, FastDiv by_groups, FastDiv by_quads, uint32_t units)
{
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const uint32_t unit = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= units) return;
    const KvUnit u = kv_unit(unit, c.heads, by_heads, groups, by_groups);
    bool bad_len;
    const KvSeq q = kv_seq(c, u.b, &bad_len);
    if (bad_len && lane == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    const int first = q.len - q.n;                  // the first token wanted
    const int g = (first >> 4) + u.j, t0 = 16 * g;  // this group's first token
    float* out = u.which ? v_out : k_out;
    if (q.n == 0 || t0 >= q.len || !out) return;
    const int page = kv_page(c, u.b, t0 >> c.log_page);
    if (page < 0) {
        if (lane == 0) kv_flag(c.err, GBX_KV_BAD_PAGE);
        return;
    }
    const int hd = c.hd;
    const int64_t ph = (int64_t)page * c.heads + u.h;
    const float s = (u.which ? c.vs : c.ks)[ph];
    const int8_t* p = (u.which ? c.v : c.k) + (ph << c.log_page) * hd + (t0 & ((1 << c.log_page) - 1)) * hd;
    float* o = out + ((int64_t)u.b * c.S + t0 - first) * ld + (int64_t)u.h * hd;   // row of token t0
    const int lo = max(0, first - t0), hi = min(16, q.len - t0);                  // the group's tokens wanted
    if (u.which) {
        for (int col = lane; col < hd; col += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(p + col * 16);
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
            float* to = o + col;
#pragma unroll
            for (int t = 0; t < 16; ++t, to += ld)
                if (t >= lo && t < hi) *to = (float)(int8_t)(x[t >> 2] >> (8 * (t & 3))) * s;
        }
    } else {
        // 128 values at a time: 8 x 16 columns are 4 loads of a lane ahead of their stores
        const int quads = hd >> 2, all = 16 * quads;
        for (int e0 = lane; e0 < all; e0 += 128) {
            char4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e0 + 32 * i < all) w[i] = *reinterpret_cast<const char4*>(p + 4 * (e0 + 32 * i));   // codes of a group are contiguous
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = e0 + 32 * i, t = (int)fast_div(e, by_quads), c4 = (e - t * quads) * 4;
                if (e >= all || t < lo || t >= hi) continue;
                float* to = o + t * ld + c4;
                const float4 f = make_float4(w[i].x * s, w[i].y * s, w[i].z * s, w[i].w * s);
                if (VEC) {
                    *reinterpret_cast<float4*>(to) = f;
                } else {
                    to[0] = f.x;
                    to[1] = f.y;
                    to[2] = f.z;
                    to[3] = f.w;
                }
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
    int64_t page_bytes;    // heads * page * hd, a multiple of 256, at most 2^30
    int64_t pages;
    int heads, layers;
    int32_t* err;
};

// One CTA per (pair, layer, K or V) and, where those are fewer than four to an
// SM, part of the page: 600 pages of 24 layers in 287 us, 6.6 TB/s, two pages of 5 in
// 2.8 (8.2 whole).  A page of a layer is one contiguous run of bytes.  Before it stores, the CTA looks its target up among
// the earlier targets and, where pages move within one pool, all sources (n words each, from L2):
// a pair that would race with another is left out, by every CTA alike.
__global__ void __launch_bounds__(256)
kv_copy_kernel(const KvPool c, const KvPool t, const int32_t* src, const int32_t* dst, int n)
{
    grid_dependency_wait();
    const bool within = c.k == t.k;
    const int i = blockIdx.x, layer = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int from = src[i], to = dst[i];
    const bool first = blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0;
    if ((uint64_t)(int64_t)from >= (uint64_t)c.pages || (uint64_t)(int64_t)to >= (uint64_t)t.pages) {
        if (first) kv_flag(c.err, GBX_KV_BAD_PAGE);
        return;
    }
    if (within && from == to) return;
    bool clash = false;
    for (int j = threadIdx.x; j < n; j += 256) clash |= (within && src[j] == to) | (j < i && dst[j] == to);
    if (__syncthreads_or(clash)) {
        if (first) kv_flag(c.err, GBX_KV_BAD_PAIR);
        return;
    }
    const uint4* s = reinterpret_cast<const uint4*>((which ? c.v : c.k) + ((int64_t)layer * c.pages + from) * c.page_bytes);
    uint4* d = reinterpret_cast<uint4*>((which ? t.v : t.k) + ((int64_t)layer * t.pages + to) * c.page_bytes);
    const int words = (int)(c.page_bytes >> 4), part = (words + (int)gridDim.z - 1) / (int)gridDim.z;
    const int end = min(words, ((int)blockIdx.z + 1) * part);
#pragma unroll 4
    for (int e = (int)blockIdx.z * part + threadIdx.x; e < end; e += 256) d[e] = s[e];
    if (blockIdx.z) return;
    const float* ss = (which ? c.vs : c.ks) + ((int64_t)layer * c.pages + from) * c.heads;
    float* ds = (which ? t.vs : t.ks) + ((int64_t)layer * t.pages + to) * c.heads;
    for (int e = threadIdx.x; e < c.heads; e += 256) ds[e] = ss[e];
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
    KvLayer c = {};
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
    if (units > 0x7fffffffLL - 8) return set_error(GBX_ERANGE, "gbx_kv_append: B=%d S=%d heads=%d", B, S, c.heads);
    KvAppend a;
    a.c = c;
    a.r.hi[0] = k_hi;
    a.r.hi[1] = v_hi;
    a.r.lo[0] = k_lo;
    a.r.lo[1] = v_lo;
    a.r.ld = ld;
    a.by_heads = make_fastdiv(c.heads);
    a.by_blocks = make_fastdiv(blocks);
    a.by_quads = make_fastdiv(c.hd / 4);
    a.blocks = blocks;
    a.units = (uint32_t)units;
    const bool vec = aligned16(k_hi) && aligned16(v_hi) && aligned16(k_lo) && aligned16(v_lo) && ld % 4 == 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // Whole pages pay for a CTA each: 256 rows of 25 heads x 64 at 16 rows a sequence and
    // 64 to a page take 13 us by rows and 27 by pages, at 32 rows 26 and 28; 64 rows at 16 to a
    // page 34 and 22, 8 prompts of 1024 rows at 64 101 and 33.
    if (S < 32 || S < P) {
        const dim3 grid((unsigned)((units + 7) / 8));
        if (vec) launch_row_kernel(kv_append_kernel<true>, grid, dim3(256), 0, s, a);
        else launch_row_kernel(kv_append_kernel<false>, grid, dim3(256), 0, s, a);
    } else {
        const dim3 block((unsigned)(32 * (P / 16) * (c.hd > 64 ? 2 : 1)));
        if (vec) launch_row_kernel(kv_append_pages_kernel<true>, dim3((unsigned)units), block, 0, s, a);
        else launch_row_kernel(kv_append_pages_kernel<false>, dim3((unsigned)units), block, 0, s, a);
    }
    return check_launch("gbx_kv_append");
}

extern "C" int gbx_kv_read(const gbx_kv_cache* cache_host, int layer, const int32_t* table, int max_pages,
                           const int32_t* kv_len, const int32_t* n, int B, int S, float* k_out, float* v_out,
                           int64_t ld, int* err_flag, gbx_stream_t stream)
{
    KvLayer c = {};
    if (int rc = kv_layer(cache_host, layer, table, max_pages, kv_len, n, B, S, err_flag, "gbx_kv_read", &c)) return rc;
    if (B == 0 || S == 0 || (!k_out && !v_out)) return GBX_OK;
    if (ld < (int64_t)c.heads * c.hd) return set_error(GBX_EINVAL, "gbx_kv_read: ld=%lld < heads*hd", (long long)ld);
    // 16-token groups that S tokens can touch
    const int64_t touched = ((int64_t)S + 30) / 16, most = (int64_t)max_pages << (c.log_page - 4);
    const int groups = (int)(touched < most ? touched : most);
    const int64_t units = (int64_t)B * groups * 2 * c.heads;
    if (units > 0x7fffffffLL - 8) return set_error(GBX_ERANGE, "gbx_kv_read: B=%d S=%d heads=%d", B, S, c.heads);
    const bool vec = aligned16(k_out) && ld % 4 == 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((units + 7) / 8));
    const FastDiv by_heads = make_fastdiv(c.heads), by_groups = make_fastdiv(groups), by_quads = make_fastdiv(c.hd / 4);
    if (vec)
        launch_row_kernel(kv_read_kernel<true>, grid, dim3(256), 0, s, c, k_out, v_out, ld, by_heads, groups, by_groups,
                          by_quads, (uint32_t)units);
    else
        launch_row_kernel(kv_read_kernel<false>, grid, dim3(256), 0, s, c, k_out, v_out, ld, by_heads, groups, by_groups,
                          by_quads, (uint32_t)units);
    return check_launch("gbx_kv_read");
}

namespace gbx {

static KvPool kv_pool(const gbx_kv_cache& h, int* err)
{
    KvPool c;
    c.k = h.k;
    c.v = h.v;
    c.ks = h.k_scale;
    c.vs = h.v_scale;
    c.page_bytes = (int64_t)h.heads * h.page * h.hd;
    c.pages = h.pages;
    c.heads = h.heads;
    c.layers = h.layers;
    c.err = err;
    return c;
}

int kv_copy_across(const gbx_kv_cache* from, const gbx_kv_cache* to, const int32_t* src, const int32_t* dst, int n, int* err_flag,
                   gbx_stream_t stream)
{
    const KvPool c = kv_pool(*from, err_flag);
    DeviceInfo di;
    if (device_info(&di) != GBX_OK) return GBX_ECUDA;
    int64_t parts = 4 * (int64_t)di.sm_count / ((int64_t)n * c.layers * 2), most = c.page_bytes / 4096;   // 256 x 16 bytes
    if (parts > most) parts = most;
    if (parts < 1) parts = 1;
    if (parts > 65535) parts = 65535;
    launch_row_kernel(kv_copy_kernel, dim3((unsigned)n, (unsigned)c.layers * 2, (unsigned)parts), dim3(256), 0,
                      reinterpret_cast<cudaStream_t>(stream), c, kv_pool(*to, err_flag), src, dst, n);
    return check_launch("gbx_kv_copy_pages");
}

}  // namespace gbx

extern "C" int gbx_kv_copy_pages(const gbx_kv_cache* cache_host, const int32_t* src, const int32_t* dst, int n,
                                 int* err_flag, gbx_stream_t stream)
{
    if (int rc = kv_check_cache(cache_host, "gbx_kv_copy_pages")) return rc;
    if (n < 0) return set_error(GBX_EINVAL, "gbx_kv_copy_pages: n=%d", n);
    if (n == 0) return GBX_OK;
    if (!src || !dst) return set_error(GBX_EINVAL, "gbx_kv_copy_pages: null pointer");
    return kv_copy_across(cache_host, cache_host, src, dst, n, err_flag, stream);
}
