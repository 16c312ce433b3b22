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
//   - a weight times its page's value scale, relative to the largest such
//     product of its row among the step's 64 tokens: unsigned digits,
//     mma.m16n8k32.u8.s8, exact.
// No code is converted (five instructions per four codes in an f16 form), and
// no sum inside the tensor cores is rounded.  A tile's 16 rows are 8 query
// rows: rows 0-7 hold digit 0 and rows 8-15 digit 1 of one instruction, a
// second one holds digit 2 (for 16 query rows: their digits 2 side by side),
// so the thread that holds a row's digit-0 sum holds the others.  The integer
// accumulators start at the bits of 1.5 2^23: the sums, below 2^22 in size,
// are then read as floats.
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
// that are used once, where a tcgen05 tile wants 128 rows.  256 sequences x 25
// heads x 2048 tokens take 255 us (6.6 TB/s, the measured copy rate) in a burst
// and 309 under the power cap, where the lower clock brings the arithmetic (243
// us from L2) near the copies; 2 x 8 heads x 120,001 tokens of width 128 with 4
// query heads each take 88 to 94 us (5.6 to 5.2 TB/s).
//
// A cluster of CTAs shares one (sequence, key head, row block): its warps take
// the 64-token steps in turn and meet in shared memory, the CTAs through
// distributed shared memory.  Where that leaves the GPU idle (few heads, a
// long cache) several clusters share the unit and meet in the workspace.
//
// Every wait for a copy is bounded (1 s): a warp that gives up, as a whole, stops
// its steps, waits (bounded) for the copies it has in flight, and its rows come
// out as NaN with GBX_LINEAR_TIMEOUT in the error flag.
#include <atomic>
#include <mutex>
#include <type_traits>

#include "kv_cache.cuh"
#include "tcgen05.cuh"
#include "tf32.cuh"

namespace gbx {

constexpr int kAcTile = 64;      // tokens per warp and step
constexpr int kAcMaxCluster = 8;
constexpr float kAcMagicF = 12582912.0f;        // 1.5 * 2^23, bits 0x4b400000
// The largest x whose balanced digits fit in 8 bits is 0x7f7f7f = 8355711; a row's
// largest entry becomes this, to a relative 2^-22.
constexpr float kAcQTop = 8355704.0f;
// A weight is 2^(x - max + 23 - 2^-19): just below 2^23 at most, so that adding 2^23
// leaves it, rounded, in the low 23 bits of the float.
constexpr float kAcPOff = 22.99999809265137f;
// A row's sums of digits and codes reach 2^23 times the values' own; held with this
// factor they stay finite for values up to 2^118 in size, and lose nothing of the
// smallest scale there is (2^-107).  The scales are read with it, and the weights'
// sum gets it after the last step, so that it leaves with the quotient.
constexpr float kAcDown = 1.9073486328125e-6f;    // 2^-19
constexpr float kAcRoom = 1.00000762939453125f;   // 1 + 2^-17

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
    int G;            // query heads per key head
    int nrb;          // row blocks per (sequence, key head)
    int nsplit;       // clusters per unit
    FastDiv by_heads, by_nrb, by_g, by_nsplit, by_hd;
    int vec, vec_out; // the rows of q, of out and out_lo are 16-byte aligned
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

// Digits 0, 1 and 2 of four 24-bit numbers, each digit's four bytes in one word.
__device__ __forceinline__ void ac_digits(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t& d0, uint32_t& d1, uint32_t& d2)
{
    const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
    d0 = __byte_perm(a, b, 0x5410);
    d1 = __byte_perm(a, b, 0x7632);
    d2 = __byte_perm(__byte_perm(w0, w1, 0x0062), __byte_perm(w2, w3, 0x0062), 0x5410);
}

// A bounded wait of a whole warp, and one verdict for it.  Every lane polls and
// reads its own clock and *abort, so some can see the phase complete that others
// have just given up on; a warp that went two ways from here would wait for good
// at its next vote or shuffle.
__device__ __forceinline__ bool ac_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint64_t limit_ns)
{
    return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort, limit_ns));
}

__device__ __forceinline__ uint4 ac_lds(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

// Constants that instructions take from registers: the accumulators' start, the
// zero digits, and pairs for the packed fp32 instructions.  Opaque, so that the
// compiler holds them in registers of their own instead of setting them up
// before every use.
struct AcConst {
    uint32_t c[4], z[2];
    float2 less, less257, less65793, by, by2, two23;
    __device__ __forceinline__ static float reg(float x)
    {
        float y;
        asm volatile("mov.f32 %0, %1;" : "=f"(y) : "f"(x));
        return y;
    }
    __device__ __forceinline__ AcConst()
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.u32 %0, 0x4b400000;" : "=r"(c[i]));
#pragma unroll
        for (int i = 0; i < 2; ++i) asm volatile("mov.u32 %0, 0;" : "=r"(z[i]));
        less = make_float2(reg(-kAcMagicF), reg(-kAcMagicF));
        by = make_float2(reg(256.0f), reg(256.0f));
        less257 = make_float2(reg(-257.0f * kAcMagicF), reg(-257.0f * kAcMagicF));
        less65793 = make_float2(reg(-65793.0f * kAcMagicF), reg(-65793.0f * kAcMagicF));
        by2 = make_float2(reg(65536.0f), reg(65536.0f));
        two23 = make_float2(reg(8388608.0f), reg(8388608.0f));
    }
};

// 65536 s2 + 256 s1 + s0 of accumulators that started at 0x4b400000, two
// neighbouring columns at a time (packed fp32, two lanes an instruction).  f_i =
// M + s_i with M = 1.5 2^23.  For the weights (U) M leaves s2 before the sum, so
// that only the sum's own roundings are left.  For the scores it leaves with one
// constant, -65793 M; that rounds to a multiple of 256 where the query's own
// rounding already cost about 500.
template <bool U>
__device__ __forceinline__ float2 ac_join(uint32_t s0, uint32_t t0, uint32_t s1, uint32_t t1, uint32_t s2, uint32_t t2, const AcConst& k)
{
    const float2 f0 = make_float2(__uint_as_float(s0), __uint_as_float(t0));
    const float2 f1 = make_float2(__uint_as_float(s1), __uint_as_float(t1));
    const float2 f2 = make_float2(__uint_as_float(s2), __uint_as_float(t2));
    if (U) return __fadd2_rn(__ffma2_rn(__fadd2_rn(f2, k.less), k.by2, __ffma2_rn(f1, k.by, k.less257)), f0);
    return __fadd2_rn(__ffma2_rn(f1, k.by, __ffma2_rn(f2, k.by2, k.less65793)), f0);
}

// 32-column blocks of a head, in pairs: a lane's 16 key bytes feed two.
constexpr int ac_chunks(int hd) { return hd > 64 ? 4 : 2; }
// Bytes between the 16-token groups of a slot.
constexpr int ac_pitch(int hd) { return 16 * hd + 32; }

// Digits of RT tiles of 8 rows.  d0, d1: [rt][m][2] (the two A registers of an
// 8-token or 8-column half), d2 likewise.
template <int RT, int M>
struct AcDigits {
    uint32_t d0[RT][M][2], d1[RT][M][2], d2[RT][M][2];
};

// s[rt]: this lane's row of tile rt against its two columns of one n8 group,
// whose B operands are the 16 bytes b[0], b[1], ..
template <bool U, int RT, int M>
__device__ __forceinline__ void ac_dot(float2 (&s)[RT], const AcDigits<RT, M>& a, const uint4* b, const AcConst& k)
{
    uint32_t x[RT][4], y[4];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const uint4 w = b[m >> 1];
        const uint32_t b0 = m & 1 ? w.z : w.x, b1 = m & 1 ? w.w : w.y;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (m == 0) ac_mma<U>(x[rt], a.d0[rt][m][0], a.d1[rt][m][0], a.d0[rt][m][1], a.d1[rt][m][1], b0, b1, k.c[0], k.c[1], k.c[2], k.c[3]);
            else ac_mma<U>(x[rt], a.d0[rt][m][0], a.d1[rt][m][0], a.d0[rt][m][1], a.d1[rt][m][1], b0, b1, x[rt][0], x[rt][1], x[rt][2], x[rt][3]);
        }
        const uint32_t z0 = RT == 2 ? a.d2[RT - 1][m][0] : k.z[0], z1 = RT == 2 ? a.d2[RT - 1][m][1] : k.z[1];
        if (m == 0) ac_mma<U>(y, a.d2[0][m][0], z0, a.d2[0][m][1], z1, b0, b1, k.c[0], k.c[1], k.c[2], k.c[3]);
        else ac_mma<U>(y, a.d2[0][m][0], z0, a.d2[0][m][1], z1, b0, b1, y[0], y[1], y[2], y[3]);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        s[rt] = ac_join<U>(x[rt][0], x[rt][1], x[rt][2], x[rt][3], y[2 * rt], y[2 * rt + 1], k);
    }
}

// The unit's rows.  Row r of a unit is call row i = r / G of query head h*G + r
// % G (the call row outermost, so that a block's rows see nearly the same keys).
struct AcUnit {
    int b, h, r0, rows;
    KvSeq seq;
};

__device__ __forceinline__ AcUnit ac_unit(const AcArgs& a, uint32_t unit, int R, bool* bad_len)
{
    AcUnit u;
    const uint32_t w = fast_div(unit, a.by_heads);
    u.h = (int)(unit - w * a.c.heads);
    u.b = (int)fast_div(w, a.by_nrb);
    u.seq = kv_seq(a.c, u.b, bad_len);
    u.r0 = (a.nrb - 1 - (int)(w - u.b * a.nrb)) * R;   // the rows that see most first
    u.rows = min(R, u.seq.n * a.G - u.r0);   // valid rows of this block, if positive
    return u;
}

// Where row r of the unit lies in q or out, but for the column.
__device__ __forceinline__ int64_t ac_row(const AcArgs& a, const AcUnit& u, int r, int64_t ld)
{
    const int rr = u.r0 + r, i = (int)fast_div(rr, a.by_g);
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

// Four neighbouring columns of an output row: acc / sum, 0 for a row that saw nothing.
__device__ __forceinline__ void ac_store4(const AcArgs& a, int64_t at, float4 acc, float sum)
{
    const float4 v = sum == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                 : make_float4(acc.x / sum, acc.y / sum, acc.z / sum, acc.w / sum);
    if (a.vec_out) {
        if (a.out_lo) {
            float4 vh, vl;
            split4(v, vh, vl);
            *reinterpret_cast<float4*>(a.out + at) = vh;
            *reinterpret_cast<float4*>(a.out_lo + at) = vl;
        } else {
            *reinterpret_cast<float4*>(a.out + at) = v;
        }
    } else {
        ac_store(a, at, v.x);
        ac_store(a, at + 1, v.y);
        ac_store(a, at + 2, v.z);
        ac_store(a, at + 3, v.w);
    }
}

// The query digits of rows base + 8 rt + n of the unit, the factor qs that turns
// a code sum into log2(e) q.c / scale, and the keys each row sees.
template <int HD, int RT>
__device__ __forceinline__ void ac_queries(const AcArgs& a, const AcUnit& u, int base, AcDigits<RT, ac_chunks(HD)>& q, float (&qs)[RT], int (&limit)[RT])
{
    constexpr int NCH = ac_chunks(HD) / 2;
    const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = base + 8 * rt + n;
        const bool ok = r < u.rows;
        limit[rt] = ok ? u.seq.len - u.seq.n + (int)fast_div(u.r0 + r, a.by_g) + 1 : 0;
        const int64_t at = ac_row(a, u, r, a.ld);
        float x[NCH][16];
        uint32_t top = 0;   // the largest |x|, as bits: NaN and infinity on top
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
            const int col = 64 * ch + 16 * cc;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (ok && col < HD) {
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
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[ch][e]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float bad = top >= 0x7f800000u ? __int_as_float(0x7fc00000) : 0.0f;
        float big = __uint_as_float(top);
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
                    // at most 8355711 in size but for rows that are not finite, whose digits do not count
                    const float f = x[ch][4 * w + e] * lift * up;
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

// One step, first half: the scores of 64 tokens whose keys lie at kb (groups
// `pitch` bytes apart), the running maximum and sum, and the weights' digits.  ks, vs: the scales of group
// cc; seen: that group can be read.  edge: some valid
// row does not see all 64 (rows past the unit's end hold zero queries and are never stored).
// one: all of them are seen and lie in one page, whose scale is all there is.
template <int HD, int RT>
__device__ __forceinline__ void ac_scores(uint32_t kb, int t0, bool seen, bool edge, bool one, float ks, float vs,
                                          const AcDigits<RT, ac_chunks(HD)>& q, const float (&qs)[RT], const int (&limit)[RT],
                                          float (&m)[RT], float (&l)[RT], AcDigits<RT, 2>& p, float (&alpha)[RT], float (&beta)[RT],
                                          const AcConst& kc)
{
    const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
    constexpr int NCH = ac_chunks(HD) / 2, pitch = ac_pitch(HD);
    float2 s[RT][8];
    vs *= kAcDown;
    // key side: this lane's tokens are 2g + (n & 1) of group n / 2
    // columns past the head's last 16 (their query digits are 0) are read from
    // those: 16 bytes further, a slot's last token would leave the ring
    const uint32_t kp = kb + (n >> 1) * pitch + (n & 1) * HD;
    uint32_t col[NCH];
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) col[ch] = min(64 * ch + 16 * cc, HD - 16);
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        uint4 w[NCH];
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) w[ch] = ac_lds(kp + 2 * g * HD + col[ch]);
        float2 d[RT];
        ac_dot<false, RT, ac_chunks(HD)>(d, q, w, kc);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][g] = d[rt];
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float2 f = splat2(qs[rt] * ks);
        float top = -INFINITY;   // of this lane's group
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            s[rt][g] = __fmul2_rn(s[rt][g], f);
            if (edge) {
                const int t = t0 + 16 * cc + 2 * g;
                if (!seen || t >= limit[rt]) s[rt][g].x = -INFINITY;
                if (!seen || t + 1 >= limit[rt]) s[rt][g].y = -INFINITY;
            }
            top = fmaxf(fmaxf(top, s[rt][g].x), s[rt][g].y);
        }
        float mt = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float mx = fmaxf(m[rt], mt), base = mx == -INFINITY ? 0.0f : mx;
        alpha[rt] = ac_exp2(m[rt] - base);
        beta[rt] = ac_exp2(mt - base);
        m[rt] = mx;
        // the maximum is taken off first, exactly where it counts; in one addition with the
        // 23 its rounding would pass 2^-19 from |max| = 32 on (0.3 % of the time)
        const float2 less = splat2(mt == -INFINITY ? 0.0f : -mt), sub = splat2(mt == -INFINITY ? 0.0f : kAcPOff);
        // The digits are relative to the row's largest product of weight and value scale among
        // the groups it sees, so that large values it does not see, or hardly weighs, cost
        // the others no bits.  kAcRoom keeps the roundings of the two exponentials and the
        // quotient below the digits' end.  A group whose weights are all below 2^-126 of the
        // step's largest counts as none, and so does a step whose products are below 2^-107.
        // With one scale that product is the scale itself, the largest weight being 1.
        float most = vs, vr = 1.0f;
        if (!one) {
            const float part = ac_exp2(top + less.x) * vs;   // NaN of a NaN scale: not taken by the maximum
            most = fmaxf(part, __shfl_xor_sync(0xffffffffu, part, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)) * kAcRoom;
            most = most >= 1.17549435e-38f ? most : 0.0f;
            vr = most > 0.0f && part > 0.0f ? __fdividef(vs, most) : 0.0f;
        }
        float2 sum = make_float2(0.0f, 0.0f), y[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            float2 x = __fadd2_rn(__fadd2_rn(s[rt][g], less), sub);
            x = make_float2(ac_exp2(x.x), ac_exp2(x.y));
            sum = __fadd2_rn(sum, x);
            y[g] = one ? __fadd2_rn(x, kc.two23) : __ffma2_rn(x, splat2(vr), kc.two23);
        }
        // a value scale that is NaN, where the row sees its group: the sum says so
        const float seen_vs = !edge || t0 + 16 * cc < limit[rt] ? vs : 0.0f;
        l[rt] = fmaf(l[rt], alpha[rt], fmaf(seen_vs, 0.0f, sum.x + sum.y) * beta[rt]);
        beta[rt] *= most;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            ac_digits(__float_as_uint(y[2 * w].x), __float_as_uint(y[2 * w].y), __float_as_uint(y[2 * w + 1].x),
                      __float_as_uint(y[2 * w + 1].y), p.d0[rt][w >> 1][w & 1], p.d1[rt][w >> 1][w & 1], p.d2[rt][w >> 1][w & 1]);
    }
}

// Second half: the output rows, rescaled by alpha, with the 64 tokens' values at
// vb added (beta: what a sum of digits and codes stands for).
template <int HD, int RT>
__device__ __forceinline__ void ac_values(uint32_t vb, const AcDigits<RT, 2>& p, const float (&alpha)[RT],
                                          const float (&beta)[RT], float2 (&o)[RT][HD / 8], const AcConst& kc)
{
    const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
    const uint32_t vp = vb + cc * ac_pitch(HD) + n * 16;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
        const uint4 w = ac_lds(vp + 8 * j * 16);
        float2 d[RT];
        ac_dot<true, RT, 2>(d, p, &w, kc);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][j] = __ffma2_rn(o[rt][j], splat2(alpha[rt]), __fmul2_rn(d[rt], splat2(beta[rt])));
    }
}

// A warp's finished rows base .. base + 8 RT - 1.
template <int HD, int RT>
__device__ __forceinline__ void ac_rows_out(const AcArgs& a, const AcUnit& u, int base, float (&l)[RT], const float2 (&o)[RT][HD / 8])
{
    const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 1);
        l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 2);
        const int r = base + 8 * rt + n;
        if (r >= u.rows) continue;
        const int64_t at = ac_row(a, u, r, a.ld_out) + 2 * cc;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            const float2 v = l[rt] == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(o[rt][j].x / l[rt], o[rt][j].y / l[rt]);
            if (a.vec_out && !a.out_lo) {
                *reinterpret_cast<float2*>(a.out + at + 8 * j) = v;
            } else if (a.vec_out) {
                float2 h, lo;
                split_value(v.x, h.x, lo.x);
                split_value(v.y, h.y, lo.y);
                *reinterpret_cast<float2*>(a.out + at + 8 * j) = h;
                *reinterpret_cast<float2*>(a.out_lo + at + 8 * j) = lo;
            } else {
                ac_store(a, at + 8 * j, v.x);
                ac_store(a, at + 8 * j + 1, v.y);
            }
        }
    }
}

// Where the rows' partial results meet: NW partial results of R rows (one per
// warp, or one that the warps fill together) and the CTA's own after them, in
// the shared memory that held the ring.
template <int HD, int R, int NW>
struct AcMeet {
    float *o, *m, *l;   // [NW + 1][R][HD], [NW + 1][R] twice
    __device__ __forceinline__ explicit AcMeet(uint8_t* smem)
        : o(reinterpret_cast<float*>(smem)), m(o + (NW + 1) * R * HD), l(m + (NW + 1) * R)
    {
    }

    // this warp's rows base .. base + 8 RT - 1, into partial result w
    template <int RT>
    __device__ __forceinline__ void put(int w, int base, int rows, const float (&mm)[RT], float (&ll)[RT], const float2 (&oo)[RT][HD / 8])
    {
        const int lane = threadIdx.x & 31, n = lane >> 2, cc = lane & 3;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            ll[rt] += __shfl_xor_sync(0xffffffffu, ll[rt], 1);
            ll[rt] += __shfl_xor_sync(0xffffffffu, ll[rt], 2);
            const int r = base + 8 * rt + n;
            if (r < rows) {
                if (cc == 0) {
                    m[w * R + r] = mm[rt];
                    l[w * R + r] = ll[rt];
                }
#pragma unroll
                for (int j = 0; j < HD / 8; ++j) *reinterpret_cast<float2*>(o + (w * R + r) * HD + 8 * j + 2 * cc) = oo[rt][j];
            }
        }
    }

    // The partial results' sum: to the output, or with more CTAs at work on the
    // unit through the cluster's shared memory to the output or the workspace.  For
    // the few rows of the splitting kernel, one column to a thread: there the form
    // below costs the kernel's loop 40 registers (256 sequences x 25 heads x 2048
    // tokens 279 us against 255), and gains nothing.
    __device__ __forceinline__ void finish_few(const AcArgs& a, const AcUnit& u, uint32_t unit, int split, uint32_t rank, uint32_t csize, int threads)
    {
        const int nr = u.rows;
        const bool alone = csize == 1 && a.nsplit == 1;
        for (int e = threadIdx.x; e < nr * HD; e += threads) {
            const int r = e / HD, col = e - r * HD;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) mx = fmaxf(mx, m[w * R + r]);
            const float base = mx == -INFINITY ? 0.0f : mx;
            float acc = 0.0f, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = ac_exp2(m[w * R + r] - base);
                acc += f * o[(w * R + r) * HD + col];
                ll += f * l[w * R + r];
            }
            if (alone) {
                ac_store(a, ac_row(a, u, r, a.ld_out) + col, ll == 0.0f ? 0.0f : acc / ll);
            } else {
                o[(NW * R + r) * HD + col] = acc;
                if (col == 0) {
                    m[NW * R + r] = mx;
                    l[NW * R + r] = ll;
                }
            }
        }
        if (alone) return;
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        auto peer = [&](uint32_t p, const float* x) -> float {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::mapa(tc::smem_u32(x), p)) : "memory");
            return v;
        };
        for (int e = (int)rank * threads + threadIdx.x; e < nr * HD; e += (int)csize * threads) {
            const int r = e / HD, col = e - r * HD;
            float mx = -INFINITY;
            for (uint32_t p = 0; p < csize; ++p) mx = fmaxf(mx, peer(p, m + NW * R + r));
            const float base = mx == -INFINITY ? 0.0f : mx;
            float acc = 0.0f, ll = 0.0f;
            for (uint32_t p = 0; p < csize; ++p) {
                const float f = ac_exp2(peer(p, m + NW * R + r) - base);
                acc += f * peer(p, o + (NW * R + r) * HD + col);
                ll += f * peer(p, l + NW * R + r);
            }
            if (a.nsplit == 1) {
                ac_store(a, ac_row(a, u, r, a.ld_out) + col, ll == 0.0f ? 0.0f : acc / ll);
            } else {
                float* w = a.ws + ((int64_t)unit * a.nsplit + split) * (R * (HD + 2));
                w[r * HD + col] = acc;
                if (col == 0) {
                    w[R * HD + r] = mx;
                    w[R * HD + R + r] = ll;
                }
            }
        }
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    }

    // The same for many rows of several CTAs (300 rows of 12 heads over 4000 tokens: 35 us
    // against 40).  The factors that bring the partial results to one maximum are formed once
    // a row; then every thread takes four columns of a row at a time.
    __device__ __forceinline__ void finish(const AcArgs& a, const AcUnit& u, uint32_t unit, int split, uint32_t rank, uint32_t csize, int threads)
    {
        constexpr int Q = HD / 4;
        const int nr = u.rows;
        for (int r = threadIdx.x; r < nr; r += threads) {
            float mx = m[r];
#pragma unroll
            for (int w = 1; w < NW; ++w) mx = fmaxf(mx, m[w * R + r]);
            const float base = mx == -INFINITY ? 0.0f : mx;
            float ll = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = ac_exp2(m[w * R + r] - base);
                ll += f * l[w * R + r];
                m[w * R + r] = f;
            }
            m[NW * R + r] = mx;
            l[NW * R + r] = ll;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < nr * Q; e += threads) {
            const int r = e / Q, col = 4 * (e - r * Q);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < NW; ++w) acc = fma4s(*reinterpret_cast<const float4*>(o + (w * R + r) * HD + col), m[w * R + r], acc);
            *reinterpret_cast<float4*>(o + (NW * R + r) * HD + col) = acc;
        }
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        auto at = [&](uint32_t p, const float* x) { return tc::mapa(tc::smem_u32(x), p); };
        auto peer = [&](uint32_t p, const float* x) -> float {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at(p, x)) : "memory");
            return v;
        };
        // factors [csize][R] in place of the first partial results, and the sums
        float* f = o;
        for (int r = threadIdx.x; r < nr; r += threads) {
            float pm[kAcMaxCluster], pl[kAcMaxCluster];
            float mx = -INFINITY;
#pragma unroll
            for (uint32_t p = 0; p < kAcMaxCluster; ++p)
                if (p < csize) {
                    pm[p] = peer(p, m + NW * R + r);
                    pl[p] = peer(p, l + NW * R + r);
                }
#pragma unroll
            for (uint32_t p = 0; p < kAcMaxCluster; ++p)
                if (p < csize) mx = fmaxf(mx, pm[p]);
            const float base = mx == -INFINITY ? 0.0f : mx;
            float ll = 0.0f;
#pragma unroll
            for (uint32_t p = 0; p < kAcMaxCluster; ++p)
                if (p < csize) {
                    const float x = ac_exp2(pm[p] - base);
                    f[p * R + r] = x;
                    ll += x * pl[p];
                }
            m[r] = mx;
            l[r] = ll;
        }
        __syncthreads();
        float* w = a.ws + ((int64_t)unit * a.nsplit + split) * (R * (HD + 2));
        for (int e = (int)rank * threads + threadIdx.x; e < nr * Q; e += (int)csize * threads) {
            const int r = e / Q, col = 4 * (e - r * Q);
            float4 v[kAcMaxCluster];
#pragma unroll
            for (uint32_t p = 0; p < kAcMaxCluster; ++p)
                if (p < csize)
                    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                                 : "=f"(v[p].x), "=f"(v[p].y), "=f"(v[p].z), "=f"(v[p].w)
                                 : "r"(at(p, o + (NW * R + r) * HD + col))
                                 : "memory");
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t p = 0; p < kAcMaxCluster; ++p)
                if (p < csize) acc = fma4s(v[p], f[p * R + r], acc);
            if (a.nsplit == 1) {
                ac_store4(a, ac_row(a, u, r, a.ld_out) + col, acc, l[r]);
            } else {
                w[r * HD + col] = acc.x;
                w[r * HD + col + 1] = acc.y;
                w[r * HD + col + 2] = acc.z;
                w[r * HD + col + 3] = acc.w;
                if (col == 0) {
                    w[R * HD + r] = m[r];
                    w[R * HD + R + r] = l[r];
                }
            }
        }
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    }
};

// Starts the copies of steps into ring slots: called by a whole warp.
constexpr int kAcArrivals = 12;   // on a slot's barrier, each phase

template <int HD>
struct AcCopies {
    const KvLayer& c;
    const int32_t* table;   // the sequence's row
    int h, maxlim, lg16;
    uint32_t ring;
    float* scales;   // [4][2][4]: key and value scales of the four groups
    __device__ __forceinline__ AcCopies(const KvLayer& c_, const AcUnit& u, int maxlim_, uint32_t ring_, float* scales_)
        : c(c_), table(c_.table + (int64_t)u.b * c_.max_pages), h(u.h), maxlim(maxlim_), lg16(c_.log_page - 4), ring(ring_), scales(scales_)
    {
    }

    // The (page, head) of this lane's group (lane & 3) of a step; -1: the page is not in the pool, -2: past the last key.
    __device__ __forceinline__ int64_t look(int step) const
    {
        const int g = 4 * step + (threadIdx.x & 3);
        if (16 * g >= maxlim) return -2;
        const int p = table[g >> lg16];
        return (unsigned)p < (unsigned)c.pages ? (int64_t)p * c.heads + h : -1;
    }

    // The keys (which = 0) or values of a step into slot s, and with the keys
    // the groups' scales into [place], -0 standing for those of a group that
    // cannot be read.  A slot's phase is twelve arrivals: lanes 0-3's, each
    // announcing its copy's bytes, and one of each of lanes 0-7.
    __device__ __forceinline__ void issue(int which, int step, int place, int s, uint32_t bar, int64_t ph) const
    {
        const int lane = threadIdx.x & 31;
        if (lane >= 8) return;
        if (lane < 4) {
            if (ph >= 0) {
                tc::mbar_arrive_expect_tx(bar, 16u * HD);
                tc::bulk_load(ring + s * 4 * ac_pitch(HD) + lane * ac_pitch(HD),
                              (which ? c.v : c.k) + (ph << c.log_page) * HD + ((4 * step + lane) & ((1 << lg16) - 1)) * 16 * HD, 16u * HD, bar);
            } else {
                tc::mbar_arrive(bar);
                if (which == 0 && ph == -1) kv_flag(c.err, GBX_KV_BAD_PAGE);
            }
        }
        float* to = scales + place * 8 + lane;
        if (which == 0 && ph >= 0) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(to)), "l"((lane < 4 ? c.ks : c.vs) + ph) : "memory");
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
        } else {
            if (which == 0) *to = -0.0f;
            tc::mbar_arrive(bar);
        }
    }
};

// HD: head width; RT: 8-row tiles; W: warps; NS: slots of a warp's ring, each
// the keys or the values of one step; ONE: pages of 64 tokens or more, so that a
// step has one value scale.  A kernel for both asks in every step, or forms four
// groups' products where there is one scale: 2 x 512 rows over 2048 tokens take
// 60 us in pages of 64 (ONE), 61 when each step asks, 63 by products; 300 rows of
// 12 heads over 4000 tokens in pages of 16 37 (35 with weights alone as the
// largest, which loses the bits of pages with smaller values).  16 rows of width
// 32 are kept to the 128 registers that four CTAs to an SM leave (28 us against 32).
template <int HD, int RT, int W, int NS, bool ONE>
__global__ void __launch_bounds__(32 * W, HD == 32 && RT == 2 ? 4 : 0) attn_cached_kernel(const AcArgs a)
{
    grid_dependency_wait();
    constexpr int R = 8 * RT, T = 32 * W;
    extern __shared__ __align__(128) uint8_t ac_smem[];
    __shared__ uint64_t bars[W][NS];
    __shared__ float s_scale[W][4][2][4];   // of step t in [t & 3]: key and value scales of the four groups
    __shared__ int s_abort;
    const KvLayer& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cc = lane & 3;
    uint32_t rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const uint32_t cid = blockIdx.x >> (31 - __clz((int)csize));   // csize is a power of two
    const uint32_t unit = fast_div(cid, a.by_nsplit);
    const int split = (int)(cid - unit * a.nsplit);
    bool bad_len;
    const AcUnit u = ac_unit(a, unit, R, &bad_len);
    if (bad_len && threadIdx.x == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    if (u.rows <= 0) return;   // every CTA of the cluster alike

    // ---------------------------------------------------- this warp's ring
    // A slot: four groups of 16 hd bytes and 32 of padding (the groups' same
    // columns then lie in different banks).  Operation 2k is the keys of this
    // warp's k-th step, 2k + 1 its values; operation j uses slot j mod NS and
    // is started as soon as operation j - NS has been read.
    constexpr int pitch = ac_pitch(HD), slot_bytes = 4 * pitch;
    const uint32_t ring = tc::smem_u32(ac_smem) + warp * NS * slot_bytes;
    const uint32_t bar0 = tc::smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int s = 0; s < NS; ++s) tc::mbar_init(bar0 + 8 * s, kAcArrivals);
        tc::fence_mbar_init();
    }
    if (threadIdx.x == 0) s_abort = 0;
    __syncthreads();
    const int maxlim = u.seq.len - u.seq.n + (int)fast_div(u.r0 + u.rows - 1, a.by_g) + 1;   // keys the last row sees
    const int minlim = u.seq.len - u.seq.n + (int)fast_div(u.r0, a.by_g) + 1;                // and the first
    const int steps = (maxlim + kAcTile - 1) / kAcTile;
    const int stride = (int)csize * a.nsplit * W;
    const int first = (split * (int)csize + (int)rank) * W + warp;
    const AcCopies<HD> copies(c, u, maxlim, ring, &s_scale[warp][0][0][0]);
    // of this warp's k-th step
    auto look = [&](int step) { return copies.look(step); };
    auto issue = [&](int which, int k, int s, int64_t ph) { copies.issue(which, first + k * stride, k & 3, s, bar0 + 8 * s, ph); };

    // pages of steps k + 1 and k + 2 of this warp while it works on step k
    static_assert(NS == 3 || NS == 4, "the page look-ahead below is two steps");
    int64_t pg[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) pg[k] = look(first + k * stride);
    int issued = 0, read = 0;   // operations
#pragma unroll
    for (int j = 0; j < NS; ++j)
        if (first + (j >> 1) * stride < steps) {
            issue(j & 1, j >> 1, j, pg[j >> 1]);
            ++issued;
        }

    AcDigits<RT, ac_chunks(HD)> q;
    float qs[RT];
    int limit[RT];
    ac_queries<HD, RT>(a, u, 0, q, qs, limit);

    float2 o[RT][HD / 8];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) o[rt][j] = make_float2(0.0f, 0.0f);
    }

    const AcConst kc;
    bool dead = false;
    int slot = 0;            // of the next operation to be read
    uint32_t phase = 0;
    volatile int* abort = &s_abort;
    uint64_t limit_ns = a.first_wait_ns;
    auto next_slot = [&] {
        ++read;
        if (++slot == NS) {
            slot = 0;
            phase ^= 1;
        }
    };
    int k = 0;
    for (int step = first; step < steps; step += stride, ++k) {
        if (limit_ns == 0 || !ac_wait(bar0 + 8 * slot, phase, abort, limit_ns)) {
            dead = true;
            break;
        }
        limit_ns = kDeviceWaitNs;
        const float ks = s_scale[warp][k & 3][0][cc], vs = s_scale[warp][k & 3][1][cc];
        const bool seen = !(ks == 0.0f && signbit(ks));
        const int t0 = step * kAcTile;
        const bool edge = __any_sync(0xffffffffu, !seen) || t0 + kAcTile > minlim;
        AcDigits<RT, 2> p;
        float alpha[RT], beta[RT];
        const uint32_t kb = ring + slot * slot_bytes;
        if (edge) ac_scores<HD, RT>(kb, t0, seen, true, false, ks, vs, q, qs, limit, m, l, p, alpha, beta, kc);
        else ac_scores<HD, RT>(kb, t0, true, false, ONE, ks, vs, q, qs, limit, m, l, p, alpha, beta, kc);
        // the keys have been read: operation 2k + NS
        __syncwarp();
        if (NS == 3 ? step + stride < steps : step + 2 * stride < steps) {
            issue(NS == 3, k + (NS == 3 ? 1 : 2), slot, pg[NS == 3 ? 1 : 2]);
            ++issued;
        }
        next_slot();
        if (!ac_wait(bar0 + 8 * slot, phase, abort, kDeviceWaitNs)) {
            dead = true;
            break;
        }
        ac_values<HD, RT>(ring + slot * slot_bytes, p, alpha, beta, o, kc);
        // the values have been read: operation 2k + 1 + NS
        __syncwarp();
        if (step + 2 * stride < steps) {
            issue(NS != 3, k + 2, slot, pg[2]);
            ++issued;
        }
        next_slot();
        pg[1] = pg[2];
        pg[2] = look(step + 3 * stride);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] *= kAcDown;
    if (dead) {
        // the copies in flight land before anything else happens to this memory
        *abort = 1;
        for (int j = read; j < issued; ++j) tc::mbar_wait(bar0 + 8 * (j % NS), (j / NS) & 1, nullptr, kDeviceWaitNs);
        if (lane == 0) kv_flag(c.err, GBX_LINEAR_TIMEOUT);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l[rt] = __int_as_float(0x7fc00000);
    }

    // ---------------------------------------------------- the warps meet
    __syncthreads();   // the ring is done with
    AcMeet<HD, R, W> meet(ac_smem);
    meet.put(warp, 0, u.rows, m, l, o);
    __syncthreads();
    meet.finish_few(a, u, unit, split, rank, csize, T);
}

// Many rows (the next tokens of a prompt): a CTA's W warps take 16 rows each and
// go through the same steps, whose copies a warp of its own keeps in flight in
// one ring.  The int8 tensor path bounds it: 16 rows x 64 tokens of width 64 are
// 96 instructions of 8 cycles, and half as many exponentials as those take.  2 x
// 512 rows x 16 heads over 2048 tokens take 60 us with 31% of the tensor cycles
// used: two warps to a scheduler do not cover each other's dependent
// instructions.  Measured and not kept: 2 or 8 warps to a CTA (63 and 67 us),
// two CTAs that split the steps (79), the next step's scores formed beside this
// one's softmax (244 registers, 82 us).
// The launch bound is one warp more than there are, which makes the register limit
// 168: from 169 on an SM's four schedulers take 8 warps, one CTA, instead of 12
// (width 32: 1038 us with an unbounded kernel's schedule, 970 with this one).
template <int HD, int W, int NS, bool ONE>
__global__ void __launch_bounds__(32 * (W + 2), HD <= 64 ? 2 : 1) attn_cached_rows_kernel(const AcArgs a)
{
    grid_dependency_wait();
    constexpr int RT = 2, R = 8 * RT * W, T = 32 * (W + 1);
    static_assert(NS <= 6, "a step's scales are kept for four steps");
    extern __shared__ __align__(128) uint8_t ac_smem[];
    __shared__ uint64_t bars[2 * NS];
    __shared__ float s_scale[4][2][4];
    __shared__ int s_abort;
    const KvLayer& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cc = lane & 3;
    uint32_t rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    uint32_t cid;
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(cid));
    const uint32_t unit = fast_div(cid, a.by_nsplit);
    const int split = (int)(cid - unit * a.nsplit);
    bool bad_len;
    const AcUnit u = ac_unit(a, unit, R, &bad_len);
    if (bad_len && threadIdx.x == 0) kv_flag(c.err, GBX_KV_BAD_LEN);
    if (u.rows <= 0) return;
    constexpr int pitch = ac_pitch(HD), slot_bytes = 4 * pitch;
    const uint32_t ring = tc::smem_u32(ac_smem), bar0 = tc::smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (NS + s); };
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            tc::mbar_init(full(s), kAcArrivals);
            tc::mbar_init(empty(s), W);
        }
        s_abort = 0;
        tc::fence_mbar_init();
    }
    __syncthreads();
    volatile int* abort = &s_abort;
    const int before = u.seq.len - u.seq.n + 1;
    const int maxlim = before + (int)fast_div(u.r0 + u.rows - 1, a.by_g);   // keys the last row sees
    const int steps = (maxlim + kAcTile - 1) / kAcTile;
    const int stride = (int)csize * a.nsplit, first = split * (int)csize + (int)rank;

    float2 o[RT][HD / 8];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) o[rt][j] = make_float2(0.0f, 0.0f);
    }
    if (warp == W) {
        // ------------------------------------------------ the copies
        AcCopies<HD> copies(c, u, maxlim, ring, &s_scale[0][0][0]);
        int issued = 0;
        int64_t page = copies.look(first);
        for (int step = first; step < steps; step += stride) {
            const int64_t next = copies.look(step + stride);
            for (int which = 0; which < 2; ++which, ++issued) {
                const int s = issued % NS;
                if (issued >= NS && !ac_wait(empty(s), (issued / NS - 1) & 1, abort, kDeviceWaitNs)) goto stop;
                copies.issue(which, step, (issued >> 1) & 3, s, full(s), page);
                __syncwarp();
            }
            page = next;
        }
    stop:
        // every copy has landed before the CTA goes on
        for (int j = max(0, issued - NS); j < issued; ++j) tc::mbar_wait(full(j % NS), (j / NS) & 1, nullptr, kDeviceWaitNs);
    } else {
        // ------------------------------------------------ this warp's rows
        const int base = 8 * RT * warp;
        AcDigits<RT, ac_chunks(HD)> q;
        float qs[RT];
        int limit[RT];
        ac_queries<HD, RT>(a, u, base, q, qs, limit);
        const int top = min(u.rows, base + 8 * RT) - 1;   // the warp's last row, if it has one
        const int wmax = top < base ? 0 : before + (int)fast_div(u.r0 + top, a.by_g);
        const int wmin = before + (int)fast_div(u.r0 + base, a.by_g);
        const AcConst kc;
        bool dead = false;
        int k = 0, slot = 0;
        uint32_t phase = 0;
        uint64_t limit_ns = a.first_wait_ns;
        auto leave = [&] {   // this warp has read the slot
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(empty(slot));
            if (++slot == NS) {
                slot = 0;
                phase ^= 1;
            }
        };
        for (int step = first; step < steps; step += stride, ++k) {
            if (limit_ns == 0 || !ac_wait(full(slot), phase, abort, limit_ns)) {
                dead = true;
                break;
            }
            limit_ns = kDeviceWaitNs;
            const int t0 = step * kAcTile;
            const bool some = t0 < wmax;   // a step past the warp's last key is let go by
            AcDigits<RT, 2> p;
            float alpha[RT], beta[RT];
            if (some) {
                const float ks = s_scale[k & 3][0][cc], vs = s_scale[k & 3][1][cc];
                const bool seen = !(ks == 0.0f && signbit(ks));
                const bool edge = __any_sync(0xffffffffu, !seen) || t0 + kAcTile > wmin;
                const uint32_t kb = ring + slot * slot_bytes;
                if (edge) ac_scores<HD, RT>(kb, t0, seen, true, false, ks, vs, q, qs, limit, m, l, p, alpha, beta, kc);
                else ac_scores<HD, RT>(kb, t0, true, false, ONE, ks, vs, q, qs, limit, m, l, p, alpha, beta, kc);
            }
            leave();
            if (!ac_wait(full(slot), phase, abort, kDeviceWaitNs)) {
                dead = true;
                break;
            }
            if (some) ac_values<HD, RT>(ring + slot * slot_bytes, p, alpha, beta, o, kc);
            leave();
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l[rt] *= kAcDown;
        if (dead) {
            *abort = 1;
            if (lane == 0) kv_flag(c.err, GBX_LINEAR_TIMEOUT);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) l[rt] = __int_as_float(0x7fc00000);
        }
    }
    if (csize == 1 && a.nsplit == 1) {
        // nobody to meet: from the registers, 32 bytes of a row at a time.  (The
        // producer stays until its copies have landed, above.)
        if (warp < W) ac_rows_out<HD, RT>(a, u, 8 * RT * warp, l, o);
        return;
    }
    __syncthreads();   // the ring is done with
    AcMeet<HD, R, 1> meet(ac_smem);
    if (warp < W) meet.put(0, 8 * RT * warp, u.rows, m, l, o);
    __syncthreads();
    meet.finish(a, u, unit, split, rank, csize, T);
}

// Joins the nsplit partial results of each unit: one CTA per unit.
__global__ void __launch_bounds__(256) attn_cached_join_kernel(const AcArgs a, int R)
{
    grid_dependency_wait();
    const uint32_t unit = blockIdx.x;
    bool bad_len;
    const AcUnit u = ac_unit(a, unit, R, &bad_len);
    const int hd = a.c.hd;
    const int64_t part = (int64_t)R * (hd + 2);
    for (int e = threadIdx.x; e < u.rows * hd; e += 256) {
        const int r = (int)fast_div(e, a.by_hd), col = e - r * hd;
        const float* w = a.ws + (int64_t)unit * a.nsplit * part;
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
// Warps per CTA and ring slots.  Measured at 256 sequences x 25 heads x 2048 tokens
// of width 64: 256 us with 4 warps and 3 slots (4 CTAs to an SM), 257 with 2 and 3,
// 275 with 2 and 4, 290 with 4 and 4, 339 with 1 and 4; at 2 x 8 heads x 120,001
// tokens of width 128: 93 with 4 and 3, 101 with 3 and 3, 103 with 2 and 3.
constexpr int kAcWarps = 4, kAcSlots = 3;
constexpr int kAcRowWarps = 4, kAcRowSlots = 6;

// One of the kernels (by head width; 8-row tiles: 1, 2, or 8 for the rows kernel;
// ONE) and the launch that goes with it.
struct AcKernel {
    void (*fn)(AcArgs);
    int threads;
    size_t smem;
};

template <int HD, int RT>
static AcKernel ac_kernel(bool one)
{
    constexpr bool many = RT == 8;
    constexpr size_t ring = (size_t)(many ? kAcRowSlots : kAcWarps * kAcSlots) * 4 * ac_pitch(HD);
    constexpr size_t meet = sizeof(float) * (size_t)((many ? 1 : kAcWarps) + 1) * 8 * RT * (HD + 2);
    AcKernel k;
    if constexpr (many)
        k.fn = one ? attn_cached_rows_kernel<HD, kAcRowWarps, kAcRowSlots, true> : attn_cached_rows_kernel<HD, kAcRowWarps, kAcRowSlots, false>;
    else
        k.fn = one ? attn_cached_kernel<HD, RT, kAcWarps, kAcSlots, true> : attn_cached_kernel<HD, RT, kAcWarps, kAcSlots, false>;
    k.threads = 32 * (many ? kAcRowWarps + 1 : kAcWarps);
    k.smem = ring > meet ? ring : meet;
    return k;
}

static AcKernel ac_kernel_of(int hd, int rt, bool one)
{
    auto of = [rt, one](auto w) {
        constexpr int HD = decltype(w)::value;
        return rt == 1 ? ac_kernel<HD, 1>(one) : rt == 2 ? ac_kernel<HD, 2>(one) : ac_kernel<HD, 8>(one);
    };
    switch (hd) {
    case 16: return of(std::integral_constant<int, 16>());
    case 32: return of(std::integral_constant<int, 32>());
    case 48: return of(std::integral_constant<int, 48>());
    case 64: return of(std::integral_constant<int, 64>());
    case 80: return of(std::integral_constant<int, 80>());
    case 96: return of(std::integral_constant<int, 96>());
    case 112: return of(std::integral_constant<int, 112>());
    default: return of(std::integral_constant<int, 128>());
    }
}

static void ac_config(const AcKernel& k, unsigned ctas, int csize, cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr)
{
    *cfg = {};
    cfg->gridDim = dim3(ctas);
    cfg->blockDim = dim3(k.threads);
    cfg->dynamicSmemBytes = k.smem;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = (unsigned)csize;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
}

// How much of a kernel the current device holds at once, asked of the runtime
// once per kernel and device: what its registers and shared memory allow, and
// how many clusters of each size its GPCs take.
struct AcResident {
    std::atomic<bool> known{false};
    int ctas;                           // per SM
    int clusters[kAcMaxCluster + 1];   // on the GPU
};

static const AcResident* ac_resident(const AcKernel& k, int hd, int rt, bool one)
{
    constexpr int kDevices = 64;   // as device_info, which has been asked before
    static AcResident all[kDevices][8][3][2];
    static std::mutex lock;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) {
        set_error(GBX_ECUDA, "gbx_attn_cached: device %d", dev);
        return nullptr;
    }
    AcResident* r = &all[dev][hd / 16 - 1][rt == 8 ? 2 : rt - 1][one];
    if (r->known.load(std::memory_order_acquire)) return r;
    std::lock_guard<std::mutex> hold(lock);
    if (r->known.load(std::memory_order_relaxed)) return r;
    bool ok = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem) == cudaSuccess &&
              cudaOccupancyMaxActiveBlocksPerMultiprocessor(&r->ctas, k.fn, k.threads, k.smem) == cudaSuccess && r->ctas > 0;
    for (int c = 1; ok && c <= kAcMaxCluster; ++c) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr;
        ac_config(k, (unsigned)c, c, &cfg, &attr);
        ok = cudaOccupancyMaxActiveClusters(&r->clusters[c], k.fn, &cfg) == cudaSuccess;
    }
    if (!ok) {
        set_error(GBX_ECUDA, "gbx_attn_cached: occupancy: %s", cudaGetErrorString(cudaGetLastError()));
        return nullptr;
    }
    r->known.store(true, std::memory_order_release);
    return r;
}

struct AcPlan {
    int rt, nrb, csize, nsplit;
    bool one;   // a step's tokens lie in one page
    int64_t units, ws_floats;
};

// cut: units may be cut into pieces that meet in a workspace.
static int ac_plan(const gbx_kv_cache* c, int B, int S, int H, int max_pages, bool cut, AcPlan* p)
{
    const int G = H / c->heads;
    const int64_t rows = (int64_t)S * G;
    if (rows > (1 << 30)) return set_error(GBX_ERANGE, "gbx_attn_cached: %d rows of %d query heads a key head", S, G);
    DeviceInfo di;
    if (device_info(&di) != GBX_OK) return GBX_ECUDA;
    // 8 or 16 rows that the warps share, splitting the steps; from 17 on 64 rows that
    // split the warps, going through the steps together (4 x 20 rows of 4 query heads
    // to a key head of width 128 over 2000 tokens: 24 us against 32 in blocks of 16)
    p->rt = rows <= 8 ? 1 : rows <= 16 ? 2 : 8;
    p->one = c->page >= kAcTile;
    const bool many = p->rt == 8;
    const int R = 8 * p->rt, W = many ? 1 : kAcWarps;   // warps that split the steps
    const int64_t nrb = (rows + R - 1) / R;
    p->units = (int64_t)B * c->heads * nrb;
    if (nrb > 0x7fffffff || p->units * kAcMaxCluster > 0x7fffffffLL)
        return set_error(GBX_ERANGE, "gbx_attn_cached: B=%d S=%d H=%d too large", B, S, H);
    p->nrb = (int)nrb;
    // The CTAs that share a unit: as many as keep every CTA resident at once (a
    // second, partly filled wave costs more than the longer loops), a step at
    // least to every warp.  Within a cluster they meet on the chip; beyond 8 in
    // the workspace, which costs a second launch and is taken where it at least
    // doubles the CTAs.
    const int64_t steps = ((int64_t)max_pages * c->page + kAcTile - 1) / kAcTile;
    const AcResident* held = ac_resident(ac_kernel_of(c->hd, p->rt, p->one), c->hd, p->rt, p->one);
    if (!held) return GBX_ECUDA;
    const int64_t resident = (int64_t)di.sm_count * held->ctas;
    int64_t share = resident / p->units;
    if (share > (steps + W - 1) / W) share = (steps + W - 1) / W;
    p->csize = 1;
    p->nsplit = 1;
    while (p->csize < kAcMaxCluster && 2 * p->csize <= share) p->csize *= 2;
    // Rows kernels, which stay on the chip longer, also take the sizes between, where
    // the GPU holds all the units' clusters at once (64 rows over 3000 tokens: 80 units in
    // threes 36 us against 49 in twos, 42 in sixes 22.6 against 29.0 in fours; 96 in threes
    // would take 56 against 49).
    if (many)
        for (int c = kAcMaxCluster - 1; c > p->csize; --c)
            if (c <= share && p->units <= held->clusters[c]) {
                p->csize = c;
                break;
            }
    if (share >= 2 * kAcMaxCluster && cut) {
        int64_t best = 0;
        for (int cs = kAcMaxCluster; cs >= 1; cs /= 2) {
            const int64_t ns = share / cs > 64 ? 64 : share / cs;
            if (cs * ns > best) {
                best = cs * ns;
                p->csize = cs;
                p->nsplit = (int)ns;
            }
        }
    }
    p->ws_floats = p->nsplit > 1 ? p->units * p->nsplit * R * (c->hd + 2) : 0;
    return GBX_OK;
}

static int ac_launch(const AcArgs& a, const AcPlan& p, cudaStream_t s)
{
    const AcKernel k = ac_kernel_of(a.c.hd, p.rt, p.one);
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    ac_config(k, (unsigned)(p.units * p.nsplit * p.csize), p.csize, &cfg, attr);
    cfg.stream = s;
    if (pdl_enabled()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaLaunchKernelEx(&cfg, k.fn, a);
    if (p.nsplit > 1)
        launch_row_kernel(attn_cached_join_kernel, dim3((unsigned)p.units), dim3(256), 0, s, a, 8 * p.rt);
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
    if (int rc = ac_plan(cache_host, B, S, H, max_pages, true, &p)) return -rc;
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
    if (int rc = ac_plan(cache_host, B, S, H, max_pages, workspace != nullptr, &p)) return rc;
    if (workspace_floats < p.ws_floats)
        if (int rc = ac_plan(cache_host, B, S, H, max_pages, false, &p)) return rc;
    a.q_hi = q_hi;
    a.q_lo = q_lo;
    a.ld = ld;
    a.out = out;
    a.out_lo = out_lo;
    a.ld_out = ld_out;
    a.ws = workspace;
    a.qscale = (float)(1.4426950408889634 / (double)scale);
    a.G = H / a.c.heads;
    a.nrb = p.nrb;
    a.nsplit = p.nsplit;
    a.by_heads = make_fastdiv(a.c.heads);
    a.by_nrb = make_fastdiv(p.nrb);
    a.by_g = make_fastdiv(a.G);
    a.by_nsplit = make_fastdiv(p.nsplit);
    a.by_hd = make_fastdiv(a.c.hd);
    a.vec_out = aligned16(out) && aligned16(out_lo) && ld_out % 4 == 0;
    a.vec = aligned16(q_hi) && aligned16(q_lo) && ld % 4 == 0;
    a.first_wait_ns = first_wait_limit_ns();
    return ac_launch(a, p, reinterpret_cast<cudaStream_t>(stream));
}
