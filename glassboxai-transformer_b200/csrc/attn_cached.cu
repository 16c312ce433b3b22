// attn_cached.cu -- attention of a few new rows per sequence over the paged
// 8-bit key/value cache (gbx_attn_cached).  No counterpart in the reference,
// which attends over freshly computed keys and values only
// (transformer.cu:213-249).
//
//   out = sum_t w_t v_t,  w = softmax_t(q . k_t / scale),  k_t = ks c_t,  v_t = vs d_t
// with integer codes c, d in [-127, 127] and one scale per (page, head).
//
// One pass over the cache, 64 tokens (four 16-token groups, each inside one
// page) per warp and step, on mma.sync.m16n8k16 (f16 inputs, f32 sums):
//   - codes become f16 without rounding (the byte c + 128 under the exponent
//     of 1024, minus 1152), two at a time;
//   - an operand that is not a code, a query or a weight, is carried as two
//     f16 halves hi + lo (22 bits).  The tile's 16 rows are 8 query rows: rows
//     0-7 hold their hi halves, 8-15 the lo ones, so one instruction forms
//     both products and a thread that holds row r's hi sum holds its lo sum;
//   - scores and weights stay in registers: lane (n, c) = (lane / 4, lane % 4)
//     loads 16 key bytes of one token, columns 16c..16c+15, and 16 value bytes
//     of one column, the tokens of group c.  The token <-> column assignment
//     of the score tiles is chosen such that the scores a lane ends up with
//     are those of group c: its weights are the second product's A operand as
//     they lie, and the scales it needs are those of one page.
// The softmax is the online form (running maximum and sum per row; the output
// is summed in fp32 registers outside the tensor cores, 64 tokens at a time,
// and rescaled when the maximum grows).  Weights are 2^(x - m + 14), times
// their group's value scale over the tile's largest one, so that the lo half
// of a small weight keeps its bits in f16's range; the factor leaves with the
// final division.
//
// A decode step reads 2 hd bytes per token and head and does 4 hd flops per
// row with them: HBM bounds it as long as the conversions and the softmax of
// the 8 row slots, used or not, fit under the loads.  Legacy mma.sync is the
// right form here: a tile has 1 to 8 useful rows of 64 keys that are used
// once, where a tcgen05 tile would want 128 rows and a trip of every code
// through shared memory as f16.
//
// A cluster of CTAs shares one (sequence, key head, row block): its warps take
// the 64-token steps in turn and meet in shared memory, the CTAs through
// distributed shared memory.  Where that leaves the GPU idle (few heads, a
// long cache) several clusters share the unit and meet in the workspace.
#include <cuda_fp16.h>

#include "kv_cache.cuh"
#include "tf32.cuh"

namespace gbx {

constexpr int kAcWarps = 8;
constexpr int kAcThreads = 32 * kAcWarps;
constexpr int kAcTile = 64;      // tokens per warp and step
constexpr int kAcMaxCluster = 8;

struct AcArgs {
    KvLayer c;
    const float* q_hi;
    const float* q_lo;
    int64_t ld;
    float* out;
    float* out_lo;
    int64_t ld_out;
    float* ws;        // partial results of nsplit > 1
    float qscale;     // log2(e) / scale
    int H, G;         // query heads, query heads per key head
    int nrb;          // row blocks per (sequence, key head)
    int nsplit;       // clusters per unit
    int64_t units;    // B * heads * nrb
};

__device__ __forceinline__ float ac_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void ac_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four codes (bytes) as f16: (bytes 0, 1) and (bytes 2, 3).
__device__ __forceinline__ void ac_codes(uint32_t w, uint32_t& a, uint32_t& b)
{
    w ^= 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), off), q = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    a = *reinterpret_cast<uint32_t*>(&p);
    b = *reinterpret_cast<uint32_t*>(&q);
}

// (x, y) as f16 pairs hi and lo with hi + lo = x, y to 22 bits.
__device__ __forceinline__ void ac_split(float x, float y, uint32_t& hi, uint32_t& lo)
{
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ uint4 ac_ld(const int8_t* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ uint32_t ac_word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// Row r of a unit: call row i = r / G of query head h*G + r % G (the call row
// outermost, so that a block's rows see nearly the same keys).
// NCH: 64-column chunks of the head; RT: 8-row tiles.
template <int NCH, int RT>
__global__ void __launch_bounds__(kAcThreads) attn_cached_kernel(const AcArgs a)
{
    grid_dependency_wait();
    constexpr int R = 8 * RT;
    extern __shared__ __align__(16) float ac_smem[];
    const KvLayer& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
    uint32_t rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const int64_t cid = blockIdx.x / csize;
    const int split = (int)(cid % a.nsplit);
    const int64_t unit = cid / a.nsplit;
    const int h = (int)(unit % c.heads);
    const int64_t w0 = unit / c.heads;
    const int rb = (int)(w0 % a.nrb), b = (int)(w0 / a.nrb);
    const int hd = c.hd, groups8 = hd >> 3;
    bool bad_len;
    const KvSeq seq = kv_seq(c, b, &bad_len);
    if (bad_len && threadIdx.x == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    const int r0 = rb * R, rows = min(R, seq.n * a.G - r0);   // valid rows of this block, if positive

    float* s_o = ac_smem;                                  // [warps][R][hd]
    float* s_m = s_o + kAcWarps * R * hd;                  // [warps][R]
    float* s_l = s_m + kAcWarps * R;                       // [warps][R]
    float* s_co = s_l + kAcWarps * R;                      // the CTA's: [R][hd], then m[R], l[R]
    float* s_cm = s_co + R * hd;
    float* s_cl = s_cm + R;

    // every CTA of the cluster takes the same way here
    if (rows <= 0) return;

    // ---------------------------------------------------- queries
    uint32_t qf[RT][NCH][4][4];
    float qs[RT];      // turns a raw sum into x = log2(e) q.c / scale (before the key scale)
    int limit[RT];     // keys the row sees
    int maxlim = 0, minlim = 0x7fffffff;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + 8 * rt + n, i = r / a.G, g = r - i * a.G;
        const bool ok = 8 * rt + n < rows;
        limit[rt] = ok ? seq.len - seq.n + i + 1 : 0;
        const int64_t at = ((int64_t)b * c.S + i) * a.ld + (int64_t)(h * a.G + g) * hd;
        float x[NCH][16];
        float big = 0.0f;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
            const int col = 64 * ch + 16 * cc;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[ch][e] = 0.0f;
                if (ok && col < hd) x[ch][e] = a.q_hi[at + col + e] + (a.q_lo ? a.q_lo[at + col + e] : 0.0f);
                big = fmaxf(big, fabsf(x[ch][e]));
            }
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // a power of two that brings the row's largest entry to [2^13, 2^14)
        const int ex = min(max((int)(__float_as_uint(big) >> 23), 14), 254) - 127;   // big's exponent, within range
        const float up = __uint_as_float((uint32_t)(127 + 13 - ex > 254 ? 254 : 127 + 13 - ex) << 23);
        qs[rt] = a.qscale * __uint_as_float((uint32_t)(127 - 13 + ex < 1 ? 1 : 127 - 13 + ex) << 23);
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ac_split(x[ch][4 * j] * up, x[ch][4 * j + 1] * up, qf[rt][ch][j][0], qf[rt][ch][j][1]);
                ac_split(x[ch][4 * j + 2] * up, x[ch][4 * j + 3] * up, qf[rt][ch][j][2], qf[rt][ch][j][3]);
            }
    }
    {
        const int last = (r0 + rows - 1) / a.G, first = r0 / a.G;
        maxlim = seq.len - seq.n + last + 1;
        minlim = seq.len - seq.n + first + 1;
    }

    float o[RT][8 * NCH][2];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8 * NCH; ++j) o[rt][j][0] = o[rt][j][1] = 0.0f;
    }

    // ---------------------------------------------------- the cache
    const int steps = (maxlim + kAcTile - 1) / kAcTile;
    const int stride = (int)csize * a.nsplit * kAcWarps;
    const int P16 = (1 << c.log_page) >> 4;   // 16-token groups per page
    const int64_t page_bytes = (int64_t)(1 << c.log_page) * hd;
    for (int step = (split * (int)csize + (int)rank) * kAcWarps + warp; step < steps; step += stride) {
        const int t0 = step * kAcTile;
        // key side: this lane's tokens are in group n / 2; value side: group cc
        const int gk = 4 * step + (n >> 1), gv = 4 * step + cc;
        int pk = -1, pv = -1;
        if (16 * gk < maxlim) pk = kv_page(c, b, gk >> (c.log_page - 4));
        if (16 * gv < maxlim) {
            pv = kv_page(c, b, gv >> (c.log_page - 4));
            if (pv < 0) kv_flag(c.err, GBX_KV_BAD_PAGE);
        }
        float ks = 0.0f, vs = 0.0f;
        if (pv >= 0) {
            ks = c.ks[(int64_t)pv * c.heads + h];
            vs = c.vs[(int64_t)pv * c.heads + h];
        }
        // scores
        float s[RT][8][2];
        const int8_t* kp = c.k + ((int64_t)pk * c.heads + h) * page_bytes + ((gk & (P16 - 1)) * 16 + (n & 1)) * hd + 16 * cc;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            float d[RT][4];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) d[rt][0] = d[rt][1] = d[rt][2] = d[rt][3] = 0.0f;
#pragma unroll
            for (int ch = 0; ch < NCH; ++ch) {
                uint4 kv = make_uint4(0, 0, 0, 0);
                if (pk >= 0 && 64 * ch + 16 * cc < hd) kv = ac_ld(kp + 2 * g * hd + 64 * ch);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t b0, b1;
                    ac_codes(ac_word(kv, j), b0, b1);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) ac_mma(d[rt], qf[rt][ch][j], b0, b1);
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s[rt][g][0] = d[rt][0] + d[rt][2];
                s[rt][g][1] = d[rt][1] + d[rt][3];
            }
        }
        // the tile's largest value scale; a NaN scale stays in the ratio, where
        // only the rows that see its group meet it
        float vmax = fmaxf(vs, __shfl_xor_sync(0xffffffffu, vs, 1));
        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
        const float vr = vmax > 0.0f ? vs / vmax : (vs == vs ? 0.0f : vs);
        vmax = vmax > 0.0f ? vmax : 0.0f;
        uint32_t pf[RT][4][4];
        float alpha[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float f = qs[rt] * ks;
            float mx = m[rt];
#pragma unroll
            for (int g = 0; g < 8; ++g)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int t = t0 + 16 * cc + 2 * g + e;
                    s[rt][g][e] = pv >= 0 && t < limit[rt] ? s[rt][g][e] * f : -INFINITY;
                    mx = fmaxf(mx, s[rt][g][e]);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float base = mx == -INFINITY ? 0.0f : mx;
            alpha[rt] = ac_exp2(m[rt] - base);
            m[rt] = mx;
            float sum = 0.0f;
            const float vrr = t0 + 16 * cc < limit[rt] ? vr : 0.0f;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const float p0 = ac_exp2(s[rt][g][0] - base + 14.0f), p1 = ac_exp2(s[rt][g][1] - base + 14.0f);
                sum += p0 + p1;
                ac_split(p0 * vrr, p1 * vrr, pf[rt][g >> 1][(g & 1) * 2], pf[rt][g >> 1][(g & 1) * 2 + 1]);
            }
            l[rt] = l[rt] * alpha[rt] + sum;
        }
        // values
        const int8_t* vp = c.v + ((int64_t)pv * c.heads + h) * page_bytes + ((gv & (P16 - 1)) * hd + n) * 16;
#pragma unroll
        for (int j = 0; j < 8 * NCH; ++j) {
            if (j >= groups8) break;
            uint4 vv = make_uint4(0, 0, 0, 0);
            if (pv >= 0) vv = ac_ld(vp + 8 * j * 16);
            float d[RT][4];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) d[rt][0] = d[rt][1] = d[rt][2] = d[rt][3] = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t b0, b1;
                ac_codes(ac_word(vv, q), b0, b1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) ac_mma(d[rt], pf[rt][q], b0, b1);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                o[rt][j][0] = o[rt][j][0] * alpha[rt] + (d[rt][0] + d[rt][2]) * vmax;
                o[rt][j][1] = o[rt][j][1] * alpha[rt] + (d[rt][1] + d[rt][3]) * vmax;
            }
        }
    }

    // ---------------------------------------------------- the CTA's warps meet
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 1);
        l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 2);
        const int r = 8 * rt + n;
        if (r < rows) {
            if (cc == 0) {
                s_m[warp * R + r] = m[rt];
                s_l[warp * R + r] = l[rt];
            }
#pragma unroll
            for (int j = 0; j < 8 * NCH; ++j)
                if (j < groups8)
                    *reinterpret_cast<float2*>(s_o + (warp * R + r) * hd + 8 * j + 2 * cc) = make_float2(o[rt][j][0], o[rt][j][1]);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * hd; e += kAcThreads) {
        const int r = e / hd, col = e - r * hd;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAcWarps; ++w) mx = fmaxf(mx, s_m[w * R + r]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float acc = 0.0f, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kAcWarps; ++w) {
            const float f = ac_exp2(s_m[w * R + r] - base);
            acc += f * s_o[(w * R + r) * hd + col];
            ll += f * s_l[w * R + r];
        }
        s_co[r * hd + col] = acc;
        if (col == 0) {
            s_cm[r] = mx;
            s_cl[r] = ll;
        }
    }
    // ---------------------------------------------------- the cluster's CTAs meet
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    const uint32_t my = (uint32_t)__cvta_generic_to_shared(s_co);
    auto peer = [&](uint32_t p, int off) -> float {
        uint32_t at;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(my + 4 * off), "r"(p));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
        return v;
    };
    for (int e = (int)rank * kAcThreads + threadIdx.x; e < rows * hd; e += (int)csize * kAcThreads) {
        const int r = e / hd, col = e - r * hd;
        float mx = -INFINITY;
        for (uint32_t p = 0; p < csize; ++p) mx = fmaxf(mx, peer(p, R * hd + r));
        const float base = mx == -INFINITY ? 0.0f : mx;
        float acc = 0.0f, ll = 0.0f;
        for (uint32_t p = 0; p < csize; ++p) {
            const float f = ac_exp2(peer(p, R * hd + r) - base);
            acc += f * peer(p, r * hd + col);
            ll += f * peer(p, R * hd + R + r);
        }
        if (a.nsplit == 1) {
            const float v = ll == 0.0f ? 0.0f : acc / ll;
            const int rr = r0 + r, i = rr / a.G, g = rr - i * a.G;
            const int64_t at = ((int64_t)b * c.S + i) * a.ld_out + (int64_t)(h * a.G + g) * hd + col;
            if (a.out_lo) {
                float vh, vl;
                split_value(v, vh, vl);
                a.out[at] = vh;
                a.out_lo[at] = vl;
            } else {
                a.out[at] = v;
            }
        } else {
            float* w = a.ws + (unit * a.nsplit + split) * (int64_t)(R * (hd + 2));
            w[r * hd + col] = acc;
            if (col == 0) {
                w[R * hd + r] = mx;
                w[R * hd + R + r] = ll;
            }
        }
    }
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Joins the nsplit partial results of each unit: one CTA per unit.
__global__ void __launch_bounds__(256) attn_cached_join_kernel(const AcArgs a, int R)
{
    grid_dependency_wait();
    const KvLayer& c = a.c;
    const int64_t unit = blockIdx.x;
    const int h = (int)(unit % c.heads);
    const int64_t w0 = unit / c.heads;
    const int rb = (int)(w0 % a.nrb), b = (int)(w0 / a.nrb), hd = c.hd;
    bool bad_len;
    const KvSeq seq = kv_seq(c, b, &bad_len);
    const int r0 = rb * R, rows = min(R, seq.n * a.G - r0);
    for (int e = threadIdx.x; e < rows * hd; e += 256) {
        const int r = e / hd, col = e - r * hd;
        const float* w = a.ws + unit * a.nsplit * (int64_t)(R * (hd + 2));
        float mx = -INFINITY;
        for (int p = 0; p < a.nsplit; ++p) mx = fmaxf(mx, w[(int64_t)p * R * (hd + 2) + R * hd + r]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float acc = 0.0f, ll = 0.0f;
        for (int p = 0; p < a.nsplit; ++p) {
            const float* x = w + (int64_t)p * R * (hd + 2);
            const float f = ac_exp2(x[R * hd + r] - base);
            acc += f * x[r * hd + col];
            ll += f * x[R * hd + R + r];
        }
        const float v = ll == 0.0f ? 0.0f : acc / ll;
        const int rr = r0 + r, i = rr / a.G, g = rr - i * a.G;
        const int64_t at = ((int64_t)b * c.S + i) * a.ld_out + (int64_t)(h * a.G + g) * hd + col;
        if (a.out_lo) {
            float vh, vl;
            split_value(v, vh, vl);
            a.out[at] = vh;
            a.out_lo[at] = vl;
        } else {
            a.out[at] = v;
        }
    }
}

// ---------------------------------------------------------------- launch
struct AcPlan {
    int rt, nch, nrb, csize, nsplit;
    int64_t units, ws_floats;
};

static int ac_plan(const gbx_kv_cache* c, int B, int S, int H, int max_pages, AcPlan* p)
{
    DeviceInfo di;
    if (device_info(&di) != GBX_OK) return GBX_ECUDA;
    const int G = H / c->heads;
    const int64_t rows = (int64_t)S * G;
    p->nch = c->hd > 64 ? 2 : 1;
    p->rt = rows > 8 && p->nch == 1 ? 2 : 1;
    const int R = 8 * p->rt;
    const int64_t nrb = (rows + R - 1) / R;
    p->units = (int64_t)B * c->heads * nrb;
    if (nrb > 0x7fffffff || p->units * kAcMaxCluster > 0x7fffffffLL)
        return set_error(GBX_ERANGE, "gbx_attn_cached: B=%d S=%d H=%d too large", B, S, H);
    p->nrb = (int)nrb;
    // two CTAs per SM; a warp has a step to itself at least
    const int64_t steps = ((int64_t)max_pages * c->page + kAcTile - 1) / kAcTile;
    const int64_t want = 2 * (int64_t)di.sm_count;
    p->csize = 1;
    while (p->csize < kAcMaxCluster && p->units * p->csize < want && (int64_t)p->csize * kAcWarps < steps) p->csize *= 2;
    p->nsplit = 1;
    if (p->csize == kAcMaxCluster)
        while (p->nsplit < 64 && p->units * p->csize * p->nsplit < want &&
               (int64_t)p->nsplit * p->csize * kAcWarps * 4 < steps)
            p->nsplit *= 2;
    p->ws_floats = p->nsplit > 1 ? p->units * p->nsplit * R * (c->hd + 2) : 0;
    return GBX_OK;
}

template <int NCH, int RT>
static int ac_launch(const AcArgs& a, const AcPlan& p, cudaStream_t s)
{
    auto k = attn_cached_kernel<NCH, RT>;
    constexpr int R = 8 * RT;
    const size_t smem = sizeof(float) * ((size_t)(kAcWarps + 1) * R * (a.c.hd + 2));
    if (smem > 48 * 1024 && cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return check_launch("gbx_attn_cached: shared-memory attribute");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.units * p.nsplit * p.csize));
    cfg.blockDim = dim3(kAcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.csize;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (pdl_enabled()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaLaunchKernelEx(&cfg, k, a);
    if (p.nsplit > 1)
        launch_row_kernel(attn_cached_join_kernel, dim3((unsigned)p.units), dim3(256), 0, s, a, R);
    return check_launch("gbx_attn_cached");
}

}  // namespace gbx

using namespace gbx;

extern "C" int64_t gbx_attn_cached_workspace(const gbx_kv_cache* cache_host, int B, int S, int H, int max_pages)
{
    if (int rc = kv_check_cache(cache_host, "gbx_attn_cached_workspace")) return -rc;
    if (B < 0 || S < 0 || max_pages < 0 || H <= 0 || H % cache_host->heads)
        return -set_error(GBX_EINVAL, "gbx_attn_cached_workspace: B=%d S=%d H=%d max_pages=%d", B, S, H, max_pages);
    if (B == 0 || S == 0) return 0;
    AcPlan p;
    if (int rc = ac_plan(cache_host, B, S, H, max_pages, &p)) return -rc;
    return p.ws_floats;
}

extern "C" int gbx_attn_cached(const gbx_kv_cache* cache_host, int layer, const float* q_hi, const float* q_lo,
                               int64_t ld, const int32_t* table, int max_pages, const int32_t* kv_len,
                               const int32_t* n_new, int B, int S, int H, float scale, float* out, float* out_lo,
                               int64_t ld_out, float* workspace, int64_t workspace_floats, int* err_flag,
                               gbx_stream_t stream)
{
    AcArgs a;
    if (int rc = kv_layer(cache_host, layer, table, max_pages, kv_len, n_new, B, S, err_flag, "gbx_attn_cached", &a.c))
        return rc;
    if (H <= 0 || H % a.c.heads)
        return set_error(GBX_EINVAL, "gbx_attn_cached: %d query heads over %d key heads", H, a.c.heads);
    if (!(scale >= 1.17549435e-38f) || scale == INFINITY)
        return set_error(GBX_EINVAL, "gbx_attn_cached: scale=%g must be a normal positive float", (double)scale);
    if (B == 0 || S == 0) return GBX_OK;
    if (!q_hi || !out) return set_error(GBX_EINVAL, "gbx_attn_cached: null pointer");
    const int64_t width = (int64_t)H * a.c.hd;
    if (ld < width || ld_out < width)
        return set_error(GBX_EINVAL, "gbx_attn_cached: ld=%lld ld_out=%lld < H*hd", (long long)ld, (long long)ld_out);
    if (workspace_floats < 0) return set_error(GBX_EINVAL, "gbx_attn_cached: workspace of %lld floats", (long long)workspace_floats);
    {
        const int64_t in_n = ((int64_t)B * S - 1) * ld + width, out_n = ((int64_t)B * S - 1) * ld_out + width;
        auto overlaps = [](const float* x, int64_t nx, const float* y, int64_t ny) {
            return x && y && x < y + ny && y < x + nx;
        };
        if (overlaps(out, out_n, q_hi, in_n) || overlaps(out, out_n, q_lo, in_n) || overlaps(out_lo, out_n, q_hi, in_n) ||
            overlaps(out_lo, out_n, q_lo, in_n) || overlaps(out, out_n, out_lo, out_n))
            return set_error(GBX_EINVAL, "gbx_attn_cached: an output overlaps the queries or the other output");
    }
    AcPlan p;
    if (int rc = ac_plan(cache_host, B, S, H, max_pages, &p)) return rc;
    if (!workspace || workspace_floats < p.ws_floats) p.nsplit = 1;
    a.q_hi = q_hi;
    a.q_lo = q_lo;
    a.ld = ld;
    a.out = out;
    a.out_lo = out_lo;
    a.ld_out = ld_out;
    a.ws = workspace;
    a.qscale = (float)(1.4426950408889634 / (double)scale);
    a.H = H;
    a.G = H / a.c.heads;
    a.nrb = p.nrb;
    a.nsplit = p.nsplit;
    a.units = p.units;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (p.nch == 1) return p.rt == 1 ? ac_launch<1, 1>(a, p, s) : ac_launch<1, 2>(a, p, s);
    return ac_launch<2, 1>(a, p, s);
}
