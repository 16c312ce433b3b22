// attn_cached.cu -- attention of a few new rows per sequence over the paged
// 8-bit key/value cache (gbx_attn_cached).  No counterpart in the reference,
// which attends over freshly computed keys and values only
// (transformer.cu:213-249).
//
//   out = sum_t w_t v_t,  w = softmax_t(q . k_t / scale),  k_t = ks c_t,  v_t = vs d_t
// with integer codes c, d in [-127, 127] and one scale per (page, head).
//
// The codes go into the tensor cores as they lie, so the other operand is
// made of 8-bit digits too, three of them (24-bit fixed point):
//   - a query row, relative to its largest entry: x = sum_k 256^k D_k with
//     signed digits, D_k . c by mma.sync.m16n8k32.s8.s8, exact;
//   - a weight, relative to the largest of its row among the step's 64
//     tokens: unsigned digits, mma.m16n8k32.u8.s8, exact.
// No code is converted (five instructions per four codes in an f16 form), and
// no sum inside the tensor cores is rounded.  A tile's 16 rows are 8 query
// rows: rows 0-7 hold digit 0 and rows 8-15 digit 1 of one instruction, a
// second one holds digit 2 (for 16 query rows: their digits 2 side by side),
// so the thread that holds a row's digit-0 sum holds the others.  The integer
// accumulators start at the bits of 1.5 2^23: the sums, below 2^22 in size,
// are then read as floats with one subtraction.
//
// One warp takes 64 tokens a step, four 16-token groups that each lie in one
// page.  Lane (n, c) = (lane / 4, lane % 4) reads 16 key bytes of one token,
// columns 16c..16c+15 of a 64-column chunk, and 16 value bytes of one column,
// the tokens of group c.  The token <-> column assignment of the score tiles
// is chosen such that the scores a lane ends up with are those of group c: its
// weights are the second product's A operand as they lie, and the scales it
// needs are those of one page.  The softmax is the online form (running
// maximum and sum per row), the output is summed in fp32 registers.
//
// A decode step reads 2 hd bytes per token and head and does 4 hd flops per
// row with them: HBM bounds it as long as the arithmetic of the 8 row slots,
// used or not, fits under the loads.  Each warp therefore runs its own ring of
// bulk copies (cp.async.bulk, one per group and operand, straight from the
// pages; 16 hd bytes each) a step or two ahead of its arithmetic.  Legacy
// mma.sync is the right form here: a tile has 1 to 8 useful rows and 64 keys
// that are used once, where a tcgen05 tile wants 128 rows.
//
// A cluster of CTAs shares one (sequence, key head, row block): its warps take
// the 64-token steps in turn and meet in shared memory, the CTAs through
// distributed shared memory.  Where that leaves the GPU idle (few heads, a
// long cache) several clusters share the unit and meet in the workspace.
//
// Every wait for a copy is bounded (1 s): a warp that gives up stops its
// steps, waits (bounded) for the copies it has in flight, and its rows come
// out as NaN with GBX_LINEAR_TIMEOUT in the error flag.
#include "kv_cache.cuh"
#include "tcgen05.cuh"
#include "tf32.cuh"

namespace gbx {

constexpr int kAcTile = 64;      // tokens per warp and step
constexpr int kAcMaxCluster = 8;
constexpr uint32_t kAcMagic = 0x4b400000u;      // 1.5 * 2^23
constexpr float kAcMagicF = 12582912.0f;
constexpr float kAcQTop = 8355711.0f;           // 0x7f7f7f: the largest x whose balanced digits fit in 8 bits
// A weight is 2^(x - max + 23 - 2^-19): just below 2^23 at most, so that adding 2^23
// leaves it, rounded, in the low 23 bits of the float.
constexpr float kAcPOff = 22.99999809265137f;

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
    int vec;          // q rows are 16-byte aligned
    uint64_t first_wait_ns;
};

__device__ __forceinline__ float ac_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// D = A B + C, int8 digits; U: A unsigned (weights) or signed (queries).
template <bool U>
__device__ __forceinline__ void ac_mma(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1, uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3)
{
    if (U)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

// 65536 s2 + 256 s1 + s0 of three accumulators that started at kAcMagic.
__device__ __forceinline__ float ac_join(uint32_t s0, uint32_t s1, uint32_t s2)
{
    const float f0 = __uint_as_float(s0) - kAcMagicF, f1 = __uint_as_float(s1) - kAcMagicF, f2 = __uint_as_float(s2) - kAcMagicF;
    return fmaf(fmaf(f2, 256.0f, f1), 256.0f, f0);
}

// Digits 0, 1 and 2 of four 24-bit numbers, each digit's four bytes in one word.
__device__ __forceinline__ void ac_digits(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t& d0, uint32_t& d1, uint32_t& d2)
{
    const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
    d0 = __byte_perm(a, b, 0x5410);
    d1 = __byte_perm(a, b, 0x7632);
    d2 = __byte_perm(__byte_perm(w0, w1, 0x0062), __byte_perm(w2, w3, 0x0062), 0x5410);
}

__device__ __forceinline__ uint4 ac_lds(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

// Digits of RT tiles of 8 rows.  d0, d1: [rt][m][2] (the two A registers of an
// 8-token or 8-column half), d2 likewise.
template <int RT, int M>
struct AcDigits {
    uint32_t d0[RT][M][2], d1[RT][M][2], d2[RT][M][2];
};

// s[rt][0..3 rows' sums]: one n8 column group against one 16-byte word group.
template <bool U, int RT, int M>
__device__ __forceinline__ void ac_dot(float (&s)[RT][2], const AcDigits<RT, M>& a, int m0, int mn, const uint4* b)
{
    uint32_t x[RT][4], y[4];
#pragma unroll
    for (int m = 0; m < mn; ++m) {
        const uint4 w = b[m >> 1];
        const uint32_t b0 = m & 1 ? w.z : w.x, b1 = m & 1 ? w.w : w.y;
        const int q = m0 + m;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (m == 0) ac_mma<U>(x[rt], a.d0[rt][q][0], a.d1[rt][q][0], a.d0[rt][q][1], a.d1[rt][q][1], b0, b1, kAcMagic, kAcMagic, kAcMagic, kAcMagic);
            else ac_mma<U>(x[rt], a.d0[rt][q][0], a.d1[rt][q][0], a.d0[rt][q][1], a.d1[rt][q][1], b0, b1, x[rt][0], x[rt][1], x[rt][2], x[rt][3]);
        }
        const uint32_t z0 = RT == 2 ? a.d2[RT - 1][q][0] : 0u, z1 = RT == 2 ? a.d2[RT - 1][q][1] : 0u;
        if (m == 0) ac_mma<U>(y, a.d2[0][q][0], z0, a.d2[0][q][1], z1, b0, b1, kAcMagic, kAcMagic, kAcMagic, kAcMagic);
        else ac_mma<U>(y, a.d2[0][q][0], z0, a.d2[0][q][1], z1, b0, b1, y[0], y[1], y[2], y[3]);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        s[rt][0] = ac_join(x[rt][0], x[rt][2], y[2 * rt]);
        s[rt][1] = ac_join(x[rt][1], x[rt][3], y[2 * rt + 1]);
    }
}

// The unit's rows.  Row r of a unit is call row i = r / G of query head h*G + r
// % G (the call row outermost, so that a block's rows see nearly the same keys).
struct AcUnit {
    int b, h, r0, rows;
    KvSeq seq;
};

__device__ __forceinline__ AcUnit ac_unit(const AcArgs& a, int64_t unit, int R, bool* bad_len)
{
    AcUnit u;
    u.h = (int)(unit % a.c.heads);
    const int64_t w = unit / a.c.heads;
    u.b = (int)(w / a.nrb);
    u.seq = kv_seq(a.c, u.b, bad_len);
    u.r0 = (int)(w % a.nrb) * R;
    u.rows = min(R, u.seq.n * a.G - u.r0);   // valid rows of this block, if positive
    return u;
}

// Where row r of the unit lies in q or out, but for the column.
__device__ __forceinline__ int64_t ac_row(const AcArgs& a, const AcUnit& u, int r, int64_t ld)
{
    const int rr = u.r0 + r, i = rr / a.G;
    return ((int64_t)u.b * a.c.S + i) * ld + (int64_t)(u.h * a.G + rr - i * a.G) * a.c.hd;
}

__device__ __forceinline__ void ac_store(const AcArgs& a, int64_t at, float v)
{
    if (a.out_lo) {
        float vh, vl;
        split_value(v, vh, vl);
        a.out[at] = vh;
        a.out_lo[at] = vl;
    } else {
        a.out[at] = v;
    }
}

// The query digits of rows base + 8 rt + n of the unit, the factor qs that turns
// a code sum into log2(e) q.c / scale, and the keys each row sees.
template <int NCH, int RT>
__device__ __forceinline__ void ac_queries(const AcArgs& a, const AcUnit& u, int base, AcDigits<RT, 2 * NCH>& q, float (&qs)[RT], int (&limit)[RT])
{
    const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3, hd = a.c.hd;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = base + 8 * rt + n;
        const bool ok = r < u.rows;
        limit[rt] = ok ? u.seq.len - u.seq.n + (u.r0 + r) / a.G + 1 : 0;
        const int64_t at = ac_row(a, u, r, a.ld);
        float x[NCH][16];
        float big = 0.0f, bad = 0.0f;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
            const int col = 64 * ch + 16 * cc;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (ok && col < hd) {
                    const float* p = a.q_hi + at + col + e;
                    const float* pl = a.q_lo ? a.q_lo + at + col + e : nullptr;
                    if (a.vec) {
                        v = *reinterpret_cast<const float4*>(p);
                        if (pl) v = add4(v, *reinterpret_cast<const float4*>(pl));
                    } else {
                        v = make_float4(p[0], p[1], p[2], p[3]);
                        if (pl) v = add4(v, make_float4(pl[0], pl[1], pl[2], pl[3]));
                    }
                }
                x[ch][e] = v.x;
                x[ch][e + 1] = v.y;
                x[ch][e + 2] = v.z;
                x[ch][e + 3] = v.w;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                big = fmaxf(big, fabsf(x[ch][e]));
                bad = fmaf(x[ch][e], 0.0f, bad);   // NaN where an entry is not finite
            }
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        bad += __shfl_xor_sync(0xffffffffu, bad, 1);
        bad += __shfl_xor_sync(0xffffffffu, bad, 2);
        // tiny rows are first brought up exactly, so that kAcQTop / big stays finite
        const float lift = big < 8.67361738e-19f ? 1.20892582e24f : 1.0f;   // 2^-60, 2^80
        big *= lift;
        const float up = big > 0.0f ? kAcQTop / big : 0.0f;
        qs[rt] = a.qscale * (big / kAcQTop) / lift + bad;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = fminf(fmaxf(x[ch][4 * w + e] * lift * up, -kAcQTop), kAcQTop);
                    // balanced digits: the bytes of x + 0x808080, each less 128
                    y[e] = (uint32_t)(__float2int_rn(f) + 0x808080);
                }
                const int m = 2 * ch + (w >> 1), hf = w & 1;
                ac_digits(y[0], y[1], y[2], y[3], q.d0[rt][m][hf], q.d1[rt][m][hf], q.d2[rt][m][hf]);
                q.d0[rt][m][hf] ^= 0x80808080u;
                q.d1[rt][m][hf] ^= 0x80808080u;
                q.d2[rt][m][hf] ^= 0x80808080u;
            }
    }
}

// One step: 64 tokens from t0 in shared memory (kb: keys, vb: values; groups
// `pitch` bytes apart) against RT tiles of 8 rows.  ks, vs: the scales of group
// cc; seen: that group can be read.  edge: some valid
// row does not see all 64 (rows past the unit's end hold zero queries and are never stored).
template <int NCH, int RT>
__device__ __forceinline__ void ac_step(uint32_t kb, uint32_t vb, int pitch, int hd, int t0, bool seen, bool edge, float ks, float vs,
                                        const AcDigits<RT, 2 * NCH>& q, const float (&qs)[RT], const int (&limit)[RT],
                                        float (&m)[RT], float (&l)[RT], float (&o)[RT][8 * NCH][2])
{
    const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
    float s[RT][8][2];
    // key side: this lane's tokens are 2g + (n & 1) of group n / 2
    const uint32_t kp = kb + (n >> 1) * pitch + (n & 1) * hd + 16 * cc;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        uint4 w[NCH];
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) w[ch] = ac_lds(kp + 2 * g * hd + 64 * ch);
        float d[RT][2];
        ac_dot<false, RT, 2 * NCH>(d, q, 0, 2 * NCH, w);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            s[rt][g][0] = d[rt][0];
            s[rt][g][1] = d[rt][1];
        }
    }
    // the step's largest value scale; a NaN scale stays in the ratio, where
    // only the rows that see its group meet it
    float vmax = fmaxf(vs, __shfl_xor_sync(0xffffffffu, vs, 1));
    vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
    const float vr = vmax > 0.0f ? __fdividef(vs, vmax) : (vs == vs ? 0.0f : vs);
    vmax = vmax > 0.0f ? vmax : 0.0f;
    AcDigits<RT, 2> p;
    float alpha[RT], beta[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float f = qs[rt] * ks;
        float mt = -INFINITY;
#pragma unroll
        for (int g = 0; g < 8; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[rt][g][e] *= f;
                if (edge && !(seen && t0 + 16 * cc + 2 * g + e < limit[rt])) s[rt][g][e] = -INFINITY;
                mt = fmaxf(mt, s[rt][g][e]);
            }
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float mx = fmaxf(m[rt], mt), base = mx == -INFINITY ? 0.0f : mx;
        alpha[rt] = ac_exp2(m[rt] - base);
        beta[rt] = ac_exp2(mt - base);
        m[rt] = mx;
        const float sub = mt == -INFINITY ? 0.0f : kAcPOff - mt;
        const float vrr = !edge || t0 + 16 * cc < limit[rt] ? vr : 0.0f;
        float sum = 0.0f;
        uint32_t y[8][2];
#pragma unroll
        for (int g = 0; g < 8; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float x = ac_exp2(s[rt][g][e] + sub);
                sum += x;
                y[g][e] = __float_as_uint(fmaf(x, vrr, 8388608.0f));
            }
        sum = fmaf(vrr, 0.0f, sum);   // a NaN scale: its digits above are no numbers, the sum says so
        l[rt] = fmaf(l[rt], alpha[rt], sum * beta[rt]);
        beta[rt] *= vmax;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            ac_digits(y[2 * w][0], y[2 * w][1], y[2 * w + 1][0], y[2 * w + 1][1], p.d0[rt][w >> 1][w & 1], p.d1[rt][w >> 1][w & 1],
                      p.d2[rt][w >> 1][w & 1]);
    }
    const uint32_t vp = vb + cc * pitch + n * 16;
#pragma unroll
    for (int j = 0; j < 8 * NCH; ++j) {
        if (8 * j >= hd) break;
        const uint4 w = ac_lds(vp + 8 * j * 16);
        float d[RT][2];
        ac_dot<true, RT, 2>(d, p, 0, 2, &w);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            o[rt][j][0] = fmaf(o[rt][j][0], alpha[rt], d[rt][0] * beta[rt]);
            o[rt][j][1] = fmaf(o[rt][j][1], alpha[rt], d[rt][1] * beta[rt]);
        }
    }
}

// NCH: 64-column chunks of the head; RT: 8-row tiles; W: warps; NS: ring stages.
template <int NCH, int RT, int W, int NS>
__global__ void __launch_bounds__(32 * W) attn_cached_kernel(const AcArgs a)
{
    grid_dependency_wait();
    constexpr int R = 8 * RT, T = 32 * W;
    extern __shared__ __align__(128) uint8_t ac_smem[];
    __shared__ uint64_t bars[W][NS];
    __shared__ float s_scale[W][NS][2][4];
    __shared__ int s_abort;
    const KvLayer& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
    uint32_t rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const int64_t cid = blockIdx.x / csize;
    const int split = (int)(cid % a.nsplit);
    const int64_t unit = cid / a.nsplit;
    bool bad_len;
    const AcUnit u = ac_unit(a, unit, R, &bad_len);
    if (bad_len && threadIdx.x == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    if (u.rows <= 0) return;   // every CTA of the cluster alike
    const int hd = c.hd;

    // ---------------------------------------------------- this warp's ring
    // a stage: 4 key groups, 4 value groups, each 16 hd bytes and 32 of padding
    // (the four groups' same columns then lie in different banks)
    const int pitch = 16 * hd + 32, stage = 8 * pitch;
    const uint32_t ring = tc::smem_u32(ac_smem) + warp * NS * stage;
    const uint32_t bar0 = tc::smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int s = 0; s < NS; ++s) tc::mbar_init(bar0 + 8 * s, 1);
        tc::fence_mbar_init();
    }
    if (threadIdx.x == 0) s_abort = 0;
    __syncthreads();
    const int maxlim = u.seq.len - u.seq.n + (u.r0 + u.rows - 1) / a.G + 1;   // keys the last row sees
    const int minlim = u.seq.len - u.seq.n + u.r0 / a.G + 1;                  // and the first
    const int steps = (maxlim + kAcTile - 1) / kAcTile;
    const int stride = (int)csize * a.nsplit * W;
    const int first = (split * (int)csize + (int)rank) * W + warp;
    const int lg16 = c.log_page - 4;
    const int64_t page_bytes = (int64_t)hd << c.log_page;
    // the page of this lane's group (lane & 3) of a step: -2 past the last key
    auto look = [&](int step) {
        const int g = 4 * step + cc;
        return step < steps && 16 * g < maxlim ? kv_page(c, u.b, g >> lg16) : -2;
    };
    // starts a step's copies into stage s; lanes 0-3 the keys, 4-7 the values
    auto issue = [&](int step, int s, int page) {
        const unsigned valid = __ballot_sync(0xffffffffu, page >= 0) & 0xffu;
        if (lane == 0) tc::mbar_arrive_expect_tx(bar0 + 8 * s, (uint32_t)__popc(valid) * 16u * (uint32_t)hd);
        __syncwarp();
        if (lane < 8 && page >= 0) {
            const int g = 4 * step + cc;
            const int8_t* src = (lane < 4 ? c.k : c.v) + ((int64_t)page * c.heads + u.h) * page_bytes + (g & ((1 << lg16) - 1)) * 16 * hd;
            tc::bulk_load(ring + s * stage + lane * pitch, src, 16u * hd, bar0 + 8 * s);
        }
        if (page == -1 && lane < 4) kv_flag(c.err, GBX_KV_BAD_PAGE);
    };
    // lane 0-3: key scale of group cc, 4-7: value scale; NaN-free 0 where there is no page.
    // The sign of a zero says whether the group can be read.
    auto scale_of = [&](int page) {
        if (page < 0) return -0.0f;
        return (lane < 4 ? c.ks : c.vs)[(int64_t)page * c.heads + u.h];
    };

    int pg = look(first);
    float sc = 0.0f;
    int issued = 0;      // steps whose copies this warp has started
    constexpr int D = NS - 1;
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const int step = first + k * stride;
        if (step < steps) {
            issue(step, k, pg);
            sc = scale_of(pg);
            pg = look(step + stride);
            if (lane < 8) s_scale[warp][k][lane >> 2][cc] = sc;
            ++issued;
        }
    }
    __syncwarp();

    AcDigits<RT, 2 * NCH> q;
    float qs[RT];
    int limit[RT];
    ac_queries<NCH, RT>(a, u, 0, q, qs, limit);

    float o[RT][8 * NCH][2];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8 * NCH; ++j) o[rt][j][0] = o[rt][j][1] = 0.0f;
    }

    bool dead = false;
    int done = 0, st = 0, last_put = -1;
    uint32_t phase = 0;
    volatile int* abort = &s_abort;
    for (int step = first; step < steps; step += stride, ++done) {
        if (last_put >= 0 && lane < 8) s_scale[warp][last_put][lane >> 2][cc] = sc;
        __syncwarp();   // and every lane has read the stage that is filled next
        last_put = -1;
        const int ahead = step + D * stride;
        if (ahead < steps) {
            const int s = st + D >= NS ? st + D - NS : st + D;
            issue(ahead, s, pg);
            sc = scale_of(pg);
            pg = look(ahead + stride);
            last_put = s;
            ++issued;
        }
        const uint64_t limit_ns = done == 0 ? a.first_wait_ns : kDeviceWaitNs;
        if (limit_ns == 0 || !tc::mbar_wait(bar0 + 8 * st, phase, abort, limit_ns)) {
            dead = true;
            break;
        }
        const float ks = s_scale[warp][st][0][cc], vs = s_scale[warp][st][1][cc];
        const bool seen = !(ks == 0.0f && signbit(ks));
        const int t0 = step * kAcTile;
        const bool edge = __any_sync(0xffffffffu, !seen) || t0 + kAcTile > minlim;
        const uint32_t kb = ring + st * stage;
        if (edge) ac_step<NCH, RT>(kb, kb + 4 * pitch, pitch, hd, t0, seen, true, ks, vs, q, qs, limit, m, l, o);
        else ac_step<NCH, RT>(kb, kb + 4 * pitch, pitch, hd, t0, true, false, ks, vs, q, qs, limit, m, l, o);
        if (++st == NS) {
            st = 0;
            phase ^= 1;
        }
    }
    if (dead) {
        // the copies in flight land before anything else happens to this memory
        *abort = 1;
        for (int k = done; k < issued; ++k) tc::mbar_wait(bar0 + 8 * (k % NS), (k / NS) & 1, nullptr, kDeviceWaitNs);
        if (lane == 0) kv_flag(c.err, GBX_LINEAR_TIMEOUT);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l[rt] = __int_as_float(0x7fc00000);
    }

    // ---------------------------------------------------- the CTA's warps meet
    __syncthreads();   // the ring is done with
    float* s_o = reinterpret_cast<float*>(ac_smem);   // [W][R][hd], then the CTA's own [R][hd]
    float* s_m = s_o + (W + 1) * R * hd;              // [W][R], then the CTA's
    float* s_l = s_m + (W + 1) * R;
    const int nr = u.rows;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 1);
        l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 2);
        const int r = 8 * rt + n;
        if (r < nr) {
            if (cc == 0) {
                s_m[warp * R + r] = m[rt];
                s_l[warp * R + r] = l[rt];
            }
#pragma unroll
            for (int j = 0; j < 8 * NCH; ++j)
                if (8 * j < hd)
                    *reinterpret_cast<float2*>(s_o + (warp * R + r) * hd + 8 * j + 2 * cc) = make_float2(o[rt][j][0], o[rt][j][1]);
        }
    }
    __syncthreads();
    const bool alone = csize == 1 && a.nsplit == 1;
    for (int e = threadIdx.x; e < nr * hd; e += T) {
        const int r = e / hd, col = e - r * hd;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[w * R + r]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float acc = 0.0f, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = ac_exp2(s_m[w * R + r] - base);
            acc += f * s_o[(w * R + r) * hd + col];
            ll += f * s_l[w * R + r];
        }
        if (alone) {
            ac_store(a, ac_row(a, u, r, a.ld_out) + col, ll == 0.0f ? 0.0f : acc / ll);
        } else {
            s_o[(W * R + r) * hd + col] = acc;
            if (col == 0) {
                s_m[W * R + r] = mx;
                s_l[W * R + r] = ll;
            }
        }
    }
    if (alone) return;
    // ---------------------------------------------------- the cluster's CTAs meet
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    auto peer = [&](uint32_t p, const float* x) -> float {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::mapa(tc::smem_u32(x), p)) : "memory");
        return v;
    };
    for (int e = (int)rank * T + threadIdx.x; e < nr * hd; e += (int)csize * T) {
        const int r = e / hd, col = e - r * hd;
        float mx = -INFINITY;
        for (uint32_t p = 0; p < csize; ++p) mx = fmaxf(mx, peer(p, s_m + W * R + r));
        const float base = mx == -INFINITY ? 0.0f : mx;
        float acc = 0.0f, ll = 0.0f;
        for (uint32_t p = 0; p < csize; ++p) {
            const float f = ac_exp2(peer(p, s_m + W * R + r) - base);
            acc += f * peer(p, s_o + (W * R + r) * hd + col);
            ll += f * peer(p, s_l + W * R + r);
        }
        if (a.nsplit == 1) {
            ac_store(a, ac_row(a, u, r, a.ld_out) + col, ll == 0.0f ? 0.0f : acc / ll);
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
    const int64_t unit = blockIdx.x;
    bool bad_len;
    const AcUnit u = ac_unit(a, unit, R, &bad_len);
    const int hd = a.c.hd;
    const int64_t part = (int64_t)R * (hd + 2);
    for (int e = threadIdx.x; e < u.rows * hd; e += 256) {
        const int r = e / hd, col = e - r * hd;
        const float* w = a.ws + unit * a.nsplit * part;
        float mx = -INFINITY;
        for (int p = 0; p < a.nsplit; ++p) mx = fmaxf(mx, w[p * part + R * hd + r]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float acc = 0.0f, ll = 0.0f;
        for (int p = 0; p < a.nsplit; ++p) {
            const float* x = w + p * part;
            const float f = ac_exp2(x[R * hd + r] - base);
            acc += f * x[r * hd + col];
            ll += f * x[R * hd + R + r];
        }
        ac_store(a, ac_row(a, u, r, a.ld_out) + col, ll == 0.0f ? 0.0f : acc / ll);
    }
}

// ---------------------------------------------------------------- launch
// Warps per CTA and ring stages: about 100 KB of ring, two CTAs to an SM.
constexpr int kAcW1 = 4, kAcS1 = 3, kAcW2 = 3, kAcS2 = 2;

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
    p->rt = rows > 8 ? 2 : 1;
    const int R = 8 * p->rt, W = p->nch == 1 ? kAcW1 : kAcW2;
    const int64_t nrb = (rows + R - 1) / R;
    p->units = (int64_t)B * c->heads * nrb;
    if (nrb > 0x7fffffff || p->units * kAcMaxCluster > 0x7fffffffLL)
        return set_error(GBX_ERANGE, "gbx_attn_cached: B=%d S=%d H=%d too large", B, S, H);
    p->nrb = (int)nrb;
    // two CTAs per SM; a warp has a step to itself at least
    const int64_t steps = ((int64_t)max_pages * c->page + kAcTile - 1) / kAcTile;
    const int64_t want = 2 * (int64_t)di.sm_count;
    p->csize = 1;
    while (p->csize < kAcMaxCluster && p->units * p->csize < want && (int64_t)p->csize * W < steps) p->csize *= 2;
    p->nsplit = 1;
    if (p->csize == kAcMaxCluster)
        while (p->nsplit < 64 && p->units * p->csize * p->nsplit < want && (int64_t)p->nsplit * p->csize * W * 4 < steps)
            p->nsplit *= 2;
    p->ws_floats = p->nsplit > 1 ? p->units * p->nsplit * R * (c->hd + 2) : 0;
    return GBX_OK;
}

template <int NCH, int RT, int W, int NS>
static int ac_launch(const AcArgs& a, const AcPlan& p, cudaStream_t s)
{
    auto k = attn_cached_kernel<NCH, RT, W, NS>;
    constexpr int R = 8 * RT;
    const size_t ring = (size_t)W * NS * 8 * (16 * a.c.hd + 32);
    const size_t meet = sizeof(float) * (size_t)(W + 1) * R * (a.c.hd + 2);
    const size_t smem = ring > meet ? ring : meet;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return check_launch("gbx_attn_cached: shared-memory attribute");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.units * p.nsplit * p.csize));
    cfg.blockDim = dim3(32 * W);
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
    a.vec = aligned16(q_hi) && aligned16(q_lo) && ld % 4 == 0;
    a.first_wait_ns = first_wait_limit_ns();
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (p.nch == 1)
        return p.rt == 1 ? ac_launch<1, 1, kAcW1, kAcS1>(a, p, s) : ac_launch<1, 2, kAcW1, kAcS1>(a, p, s);
    return p.rt == 1 ? ac_launch<2, 1, kAcW2, kAcS2>(a, p, s) : ac_launch<2, 2, kAcW2, kAcS2>(a, p, s);
}
