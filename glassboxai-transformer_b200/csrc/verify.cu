// verify.cu -- verification of drafted tokens against the target's
// distributions (gbx_verify_tokens), beside the next-token selection of
// select.cu.  No counterpart in the reference (its generate loop takes one
// token per forward, transformer.cu:986-1036).
//
// One cluster of 16 or 8 CTAs per sequence, one launch; each of its warps owns
// one run of the vocabulary.
//   A  the rows' statistics: the warp's share of every target and draft row;
//      maximum and sum of 2^((x - m) log2(e) / T) in one pass (running maximum
//      per lane).  fp32: the sum decides a test whose border is a single point.
//   B  every CTA takes the same decision from the statistics and the drafted
//      tokens' own logits: the first draft that is not accepted.
//   C  the next token by inversion of the running sum of r_j = max(p_j - q_j,
//      0) (p_j after the last draft): the two normalisers, the runs' sums, and
//      then the one run that holds the border.  A lane owns neighbouring
//      entries of its warp's run, whose exponentials stay in shared memory, so
//      a run's sum, its lanes' prefixes and the entry come from one evaluation.
//      fp64: a vocabulary has a border every few
//      1e-5 of the sum, so an error of 1e-7 in the running sum would pick a
//      neighbour every few hundred draws.
// What the CTAs tell one another they write into each other's shared memory
// before a cluster barrier, so that every read after it is local.
// At temperature <= 0.01 A finds each target row's first maximum and C is not
// needed.
//
// The fp64 exponential is table-driven (P. T. P. Tang, "Table-driven
// implementation of the exponential function in IEEE floating-point
// arithmetic", 1989): with t = 128 (x - m) / (T ln 2),
// k = rint(t) and r = t - k, e^((x - m) / T) = 2^(k/128) e^(r ln 2 / 128), the
// second factor by its Taylor polynomial of degree 4 (|r ln 2 / 128| < 0.0028:
// remainder below 1.3e-15), the 128 roots computed into shared memory by
// exp2(): ten fp64 instructions where the fp64 pipe is what bounds C.
#include <atomic>

#include "gbx_common.cuh"
#include "kv_cache.cuh"
#include "row_stats.cuh"

namespace gbx {

constexpr int kVfMaxDraft = 256;
constexpr size_t kVfStatic = 8192;   // shared memory left to the kernel's own arrays, at least
constexpr int kVfQuads = 2;      // 16-byte loads of a lane in one unit of A

// A warp's run of the vocabulary, and a lane's neighbouring entries of it (odd:
// the lanes' doubles then lie in different banks).
__host__ __device__ constexpr int vf_run(int vocab, int runs) { return (vocab + runs - 1) / runs; }
__host__ __device__ constexpr int vf_seg(int run) { return ((run + 31) / 32) | 1; }
// Dynamic shared memory: the rows' statistics, then where they fit (KEEP) the
// exponentials of each warp's run in both distributions.
constexpr size_t vf_stats(int n, int cluster, int warps) { return sizeof(float2) * (2 * n + 1) * (warps + cluster + 1); }
constexpr size_t vf_kept(int vocab, int cluster, int warps) { return sizeof(double) * 2 * warps * 32 * vf_seg(vf_run(vocab, cluster * warps)); }

struct VfArgs {
    const float* logits;
    const float* draft_logits;
    const int32_t* draft_ids;
    const int32_t* draft_len;
    int n, vocab;
    double inv_t;     // 1 / temperature
    float c2;         // log2(e) / temperature
    int greedy;
    const double* uniforms;
    int32_t* out_ids;
    int32_t* n_accepted;
    int32_t* err;
};

__device__ __forceinline__ float vf_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void vf_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void vf_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The address in CTA `rank` of the cluster of this CTA's shared memory at p.
__device__ __forceinline__ uint32_t vf_peer(const void* p, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}

__device__ __forceinline__ void vf_push(const float2* p, uint32_t rank, float2 v)
{
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(vf_peer(p, rank)), "f"(v.x), "f"(v.y) : "memory");
}

__device__ __forceinline__ void vf_push(const double* p, uint32_t rank, double v)
{
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(vf_peer(p, rank)), "d"(v) : "memory");
}

// A part of a row: x its maximum, y the sum of 2^((v - x) c2) over it; greedy:
// x the maximum (NaN where an entry is) and y the bits of its first index.
__device__ __forceinline__ float2 vf_better(float2 a, float2 b)
{
    if (a.x != a.x) return a;
    if (b.x != b.x) return b;
    return b.x > a.x || (b.x == a.x && __float_as_int(b.y) < __float_as_int(a.y)) ? b : a;
}

// Of N neighbouring lanes' parts, in a fixed tree; the same bits in each of them.
template <int N>
__device__ __forceinline__ float2 vf_reduce(float2 v, float c2, int greedy)
{
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const float2 w = make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
        v = greedy ? vf_better(v, w) : row_join(v, w, c2, [](float x) { return vf_exp2(x); });
    }
    return v;
}

// The exponential of one distribution (see the header): e^((x - m) / T) of a
// logit x; 0 below e^-700.  x - m is formed first: as one FMA with m c rounded,
// a row of nothing but the lowest float would lose its equal entries.
struct VfExp {
    double m, c;          // t = (x - m) c
    const double* root;   // 2^(i/128)
    __device__ __forceinline__ VfExp(double m_, double inv_t, const double* roots)
        : m(m_), c(inv_t * 184.6649652337873), root(roots)
    {
    }
    __device__ __forceinline__ double operator()(float x) const
    {
        const double t = ((double)x - m) * c;
        const double big = t + 6755399441055744.0;       // 1.5 2^52: k in the low word
        const double r = t - (big - 6755399441055744.0);
        const int k = __double2loint(big);
        double p = fma(r, 3.583032305400251e-11, 2.646642144433097e-08);   // (ln 2 / 128)^i / i!, i = 4, 3
        p = fma(r, p, 1.4662262387640425e-05);                             // 2
        p = fma(r, p, 0.0054152123481245725);                              // 1
        p = fma(r, p, 1.0);
        const double f = root[k & 127];
        const double e = p * __hiloint2double(__double2hiint(f) + ((k >> 7) << 20), __double2loint(f));
        return t > -129265.0 ? e : 0.0;                  // -700 in units of ln 2 / 128: the exponent stays normal
    }
};

// C: CTAs of a cluster.
// W: warps of a CTA.
enum { VF_GREEDY, VF_AGAIN, VF_KEEP };   // sampling: part C forms its exponentials again, or keeps them in shared memory
template <int C, int W, int MODE>
__global__ void __launch_bounds__(32 * W, W == 8 ? 3 : 2) verify_kernel(const VfArgs a)
{
    constexpr int kVfRuns = C * W, kVfThreads = 32 * W;
    constexpr bool GREEDY = MODE == VF_GREEDY, KEEP = MODE == VF_KEEP;
    constexpr int kVfAhead = W == 8 ? 3 : 2;   // units of A in flight
    grid_dependency_wait();
    vf_arrive();   // awaited before the first write into another CTA
    extern __shared__ __align__(16) float2 s_warp[];                                            // [rows][warps]
    __shared__ double s_root[128];
    __shared__ double s_z[2][kVfRuns], s_run[kVfRuns];
    __shared__ int s_dec;         // accepted drafts
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int64_t b = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = a.n, V = a.vocab, max_rows = 2 * n + 1;
    float2* s_part = s_warp + max_rows * W;                                              // [rows][CTAs]
    float2* s_stat = s_part + max_rows * C;                                                     // [rows]
    int len = a.draft_len ? a.draft_len[b] : n;
    const bool bad_len = len < 0 || len > n;
    if (bad_len) len = 0;
    const float* tl = a.logits + b * (n + 1) * (int64_t)V;
    const float* dl = a.draft_logits && !GREEDY ? a.draft_logits + b * (int64_t)n * V : nullptr;
    const int32_t* ids = a.draft_ids + b * n;
    // this warp's run of a row in C
    const int run = vf_run(V, kVfRuns), seg = vf_seg(run);
    const int me = (int)rank * W + warp;
    const int j0 = min(V, me * run), j1 = min(V, j0 + run);
    const int nrows = bad_len ? 0 : len + 1 + (dl ? len : 0);
    auto row = [&](int k) { return k <= len ? tl + (int64_t)k * V : dl + (int64_t)(k - len - 1) * V; };

    // ---------------------------------------------------- A
    // Here a warp's share of a row is a run of 16-byte quads, which start at the
    // row's own first aligned entry; the up to six entries around them are warp
    // 0's.  Unit u: pass u % passes (64 quads) of row u / passes, the next few
    // units' loads in flight while one is worked on.
    constexpr int N = kVfQuads, Q = 32 * N;
    const int share = ((V >> 2) + kVfRuns) / kVfRuns, passes = (share + Q - 1) / Q;
    struct Unit {
        float4 v[N];
        float x;    // one of the entries around the quads, or -inf
        int j;      // v[i] holds entries j + 128 i ..
        int jx;
    };
    auto fetch = [&](int k, int pass) {
        const float* x = row(k);
        const int head = min(V, (int)((4 - ((reinterpret_cast<uintptr_t>(x) >> 2) & 3)) & 3)), quads = (V - head) >> 2;
        const int q0 = me * share + pass * Q + lane, q1 = min(quads, (me + 1) * share);
        Unit u;
        u.j = head + 4 * q0;
        const float4* at = reinterpret_cast<const float4*>(x + head) + q0;
#pragma unroll
        for (int i = 0; i < N; ++i) u.v[i] = q0 + 32 * i < q1 ? at[32 * i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const int tail = V - head - 4 * quads;
        u.jx = lane < 4 ? lane : head + 4 * quads + lane - 4;
        u.x = me == 0 && pass == 0 && (lane < 4 ? lane < head : lane - 4 < tail) ? x[u.jx] : -INFINITY;
        return u;
    };
    int fk = 0, fp = 0;   // the unit that is fetched next
    Unit next[kVfAhead];
    auto fetch_next = [&](Unit& u) {
        if (fk < nrows) u = fetch(fk, fp);
        if (++fp == passes) {
            fp = 0;
            ++fk;
        }
    };
#pragma unroll
    for (int i = 0; i < kVfAhead; ++i) fetch_next(next[i]);
    // what B and C need from memory, asked for meanwhile
    const double u_next = GREEDY ? 0.0 : a.uniforms[b * (n + 1) + n];
    int d_mine = -1;
    float tl_mine = 0.0f, dl_mine = 0.0f;
    double u_mine = 0.0;
    if (tid < len) {
        d_mine = ids[tid];
        if (!GREEDY) u_mine = a.uniforms[b * (n + 1) + tid];
        if ((unsigned)d_mine < (unsigned)V) {
            tl_mine = tl[(int64_t)tid * V + d_mine];
            if (dl) dl_mine = dl[(int64_t)tid * V + d_mine];
        }
    }
    if (tid < 128) s_root[tid] = exp2(tid * (1.0 / 128.0));
    if (tid == 0) s_dec = len;
    float m = -INFINITY, s = 0.0f;
    int at = 0x7fffffff, k = 0, pass = 0;
    bool nan = false;
    const int units = nrows * passes;
    for (int u0 = 0; u0 < units; u0 += kVfAhead) {
        // unrolled, so that each unit in flight has registers of its own: moving
        // one that is still loading would wait for it
#pragma unroll
        for (int i = 0; i < kVfAhead; ++i) {
            if (u0 + i >= units) continue;
            const Unit& u = next[i];
            static_assert(N == 2, "as written out here");
            const float v[4 * N + 1] = {u.v[0].x, u.v[0].y, u.v[0].z, u.v[0].w, u.v[1].x, u.v[1].y, u.v[1].z, u.v[1].w, u.x};
            if (GREEDY) {
#pragma unroll
                for (int e = 0; e <= 4 * N; ++e) {
                    const int j = e == 4 * N ? u.jx : u.j + 128 * (e >> 2) + (e & 3);
                    nan |= v[e] != v[e];
                    if (v[e] > m || (v[e] == m && j < at)) {
                        m = v[e];
                        at = j;
                    }
                }
            } else {
                float bm = fmaxf(m, v[4 * N]);
#pragma unroll
                for (int e = 0; e < 4 * N; ++e) bm = fmaxf(bm, v[e]);
                // the maximum is taken off first: a mask of the lowest float times c2 would overflow
                const float base = bm == -INFINITY ? 0.0f : bm;
                const float2 by = splat2(a.c2), less = splat2(-base);
                float2 t = make_float2(vf_exp2((v[4 * N] - base) * a.c2), 0.0f);   // a NaN makes the sum NaN
#pragma unroll
                for (int e = 0; e < 4 * N; e += 2) {
                    const float2 y = __fmul2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), less), by);
                    t = __fadd2_rn(t, make_float2(vf_exp2(y.x), vf_exp2(y.y)));
                }
                s = fmaf(s, vf_exp2((m - base) * a.c2), t.x + t.y);                // m = -inf: 0
                m = bm;
            }
            fetch_next(next[i]);
            if (++pass < passes) continue;
            float2 st;
            if (GREEDY) {
                st = vf_reduce<32>(make_float2(nan ? __int_as_float(0x7fc00000) : m, __int_as_float(at)), a.c2, 1);
            } else {
                const float wm = group_max<32>(m), base = wm == -INFINITY ? 0.0f : wm;
                st = make_float2(wm, group_sum<32>(s * vf_exp2((m - base) * a.c2)));
            }
            if (lane == 0) s_warp[k * W + warp] = st;
            ++k;
            pass = 0;
            m = -INFINITY;
            s = 0.0f;
            at = 0x7fffffff;
            nan = false;
        }
    }
    __syncthreads();
    vf_wait();   // the other CTAs run
    // This CTA's part of each row, to every CTA: one lane's value to all of them,
    // since each takes part B's decision for itself and they have to agree on it.
    for (int i = tid; i < (nrows * W + 31 & ~31); i += kVfThreads) {
        const int k = i / W, w = i % W;
        float2 t = vf_reduce<W>(k < nrows ? s_warp[i] : make_float2(-INFINITY, 0.0f), a.c2, GREEDY);
        t = make_float2(__shfl_sync(0xffffffffu, t.x, 0, W), __shfl_sync(0xffffffffu, t.y, 0, W));
        if (k < nrows)
            for (uint32_t p = w; p < C; p += W) vf_push(s_part + k * C + rank, p, t);
    }
    vf_arrive();
    vf_wait();
    // the whole rows; x NaN: the row gives no distribution
    for (int i = tid; i < (nrows * C + 31 & ~31); i += kVfThreads) {
        const int k = i / C;
        float2 t = vf_reduce<C>(k < nrows ? s_part[i] : make_float2(-INFINITY, 0.0f), a.c2, GREEDY);
        if (fabsf(t.x) == INFINITY || (!GREEDY && t.y != t.y)) t.x = __int_as_float(0x7fc00000);
        if (k < nrows && i % C == 0) s_stat[k] = t;
    }
    __syncthreads();

    // ---------------------------------------------------- B
    if (tid < len) {
        const float2 st = s_stat[tid];
        const bool known = (unsigned)d_mine < (unsigned)V;
        if (!known && rank == 0) kv_flag(a.err, GBX_VERIFY_BAD_ID);
        bool ok = st.x == st.x && known;
        if (ok && GREEDY) {
            ok = d_mine == __float_as_int(st.y);
        } else if (ok) {
            double q = 1.0;
            if (dl) {
                const float2 sq = s_stat[len + 1 + tid];
                ok = sq.x == sq.x;
                if (ok) q = VfExp(sq.x, a.inv_t, s_root)(dl_mine) / (double)sq.y;
            }
            ok = ok && u_mine * q < VfExp(st.x, a.inv_t, s_root)(tl_mine) / (double)st.y;
        }
        if (!ok) atomicMin(&s_dec, tid);
    }
    __syncthreads();
    const int acc = s_dec;
    const bool rejected = acc < len;
    bool bad = bad_len;
    float2 sp = make_float2(0.0f, 0.0f), sq = sp;
    if (!bad) {
        sp = s_stat[acc];
        bad = !(sp.x == sp.x);
        if (rejected && dl) {
            sq = s_stat[len + 1 + acc];
            bad |= !(sq.x == sq.x);
        }
    }
    if (rank == 0) {
        const int next = GREEDY && !bad ? __float_as_int(sp.y) : -1;
        for (int i = tid; i <= n; i += kVfThreads)
            if (i != acc || GREEDY || bad) a.out_ids[b * (n + 1) + i] = i < acc ? ids[i] : i == acc ? next : -1;
        if (tid == 0) {
            a.n_accepted[b] = acc;
            if (bad) kv_flag(a.err, GBX_VERIFY_BAD_ROW);
        }
    }
    if (GREEDY || bad) return;   // every CTA of the cluster alike

    // ---------------------------------------------------- C
    const float* px = tl + (int64_t)acc * V;
    const float* qx = rejected && dl ? dl + (int64_t)acc * V : nullptr;
    const int hot = rejected && !dl ? ids[acc] : -1;   // a draft picked without chance
    const VfExp pexp(sp.x, a.inv_t, s_root), qexp(sq.x, a.inv_t, s_root);
    // the run's e^((x - m) / T), kept or formed again; entry i of this lane's is i of the run
    double* kept_p = reinterpret_cast<double*>(s_stat + max_rows + (max_rows & 1)) + warp * 2 * 32 * seg;
    double* kept_q = kept_p + 32 * seg;
    auto prob = [&](int i) { return KEEP ? kept_p[i] : j0 + i < j1 ? pexp(px[j0 + i]) : 0.0; };
    auto other = [&](int i) { return !qx ? 0.0 : KEEP ? kept_q[i] : j0 + i < j1 ? qexp(qx[j0 + i]) : 0.0; };
    auto sum32 = [](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    double zp = 0.0, zq = 0.0;
    for (int i = lane; i < 32 * seg; i += 128) {   // four loads of each row before their use
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = j0 + i + 32 * e;
            x[e] = j < j1 ? px[j] : -INFINITY;
            y[e] = qx && j < j1 ? qx[j] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double p = pexp(x[e]), q = qx ? qexp(y[e]) : 0.0;
            zp += p;
            zq += q;
            if (KEEP && i + 32 * e < 32 * seg) {
                kept_p[i + 32 * e] = p;
                kept_q[i + 32 * e] = q;
            }
        }
    }
    __syncwarp();
    zp = sum32(zp);
    zq = sum32(zq);
    if (lane < C) {
        vf_push(&s_z[0][me], lane, zp);
        vf_push(&s_z[1][me], lane, zq);
    }
    vf_arrive();
    vf_wait();
    // every warp adds the runs' sums in the same order
    zp = zq = 0.0;
#pragma unroll
    for (int e = 0; e < kVfRuns / 32; ++e) {
        zp += s_z[0][lane + 32 * e];
        zq += s_z[1][lane + 32 * e];
    }
    const double ip = 1.0 / sum32(zp), iq = qx ? 1.0 / sum32(zq) : 0.0;
    bool minus = rejected;
    auto weight = [&](int i) {
        // rounded products: equal p and q leave exactly nothing, and every evaluation the same
        const double p = __dmul_rn(prob(i), ip);
        if (!minus) return p;
        const double q = qx ? __dmul_rn(other(i), iq) : j0 + i == hot ? 1.0 : 0.0;
        return p > q ? __dsub_rn(p, q) : 0.0;
    };
    auto scan32 = [&](double v) {   // inclusive
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += up;
        }
        return v;
    };
    for (;;) {
        double mine_sum = 0.0;   // of this lane's entries
#pragma unroll 4
        for (int i = lane * seg; i < (lane + 1) * seg; ++i) mine_sum += weight(i);
        const double mine_incl = scan32(mine_sum), t = __shfl_sync(0xffffffffu, mine_incl, 31);
        if (lane < C) vf_push(&s_run[me], lane, t);
        vf_arrive();
        vf_wait();
        // the running sum over the runs: lane l holds kPer of them
        constexpr int kPer = kVfRuns / 32;
        double r[kPer], mine = 0.0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            r[e] = s_run[lane * kPer + e];
            mine += r[e];
        }
        const double incl = scan32(mine), all = __shfl_sync(0xffffffffu, incl, 31);
        if (!(all > 0.0) && minus) {   // p = q: of p itself (every CTA alike)
            minus = false;
            vf_arrive();               // the runs' sums have been read
            vf_wait();
            continue;
        }
        const double want = (u_next > 0.0 ? u_next : 0.0) * all;
        // the first run whose running sum passes `want`, and the sum before it
        int found = -1, any = -1;
        double before = incl - mine, at_run = 0.0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if (found < 0 && before + r[e] > want && r[e] > 0.0) {
                found = lane * kPer + e;
                at_run = before;
            }
            before += r[e];
            if (r[e] > 0.0) any = lane * kPer + e;
        }
        const unsigned who = __ballot_sync(0xffffffffu, found >= 0), some = __ballot_sync(0xffffffffu, any >= 0);
        // none (u * all rounded up to all): the last entry with any weight
        const int owner = who ? __ffs(who) - 1 : 31 - __clz(some);
        found = __shfl_sync(0xffffffffu, who ? found : any, owner);
        const double cum = __shfl_sync(0xffffffffu, at_run, owner);
        if (found != me) return;
        // the entry, and the run's last one with any weight, should rounding end the run early
        double at = cum + (mine_incl - mine_sum);
        int pick = 0x7fffffff, last = -1;
        for (int i = lane * seg; i < (lane + 1) * seg; ++i) {
            const double w = weight(i);
            at += w;
            if (w > 0.0) {
                last = j0 + i;
                if (at > want) pick = min(pick, j0 + i);
            }
        }
        pick = __reduce_min_sync(0xffffffffu, pick);
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) a.out_ids[b * (n + 1) + acc] = pick != 0x7fffffff ? pick : last;
        return;
    }
}

template <int C, int W>
static int vf_launch(const VfArgs& a, int64_t B, const DeviceInfo& di, cudaStream_t s)
{
    const size_t stats = vf_stats(a.n, C, W) + 8, kept = vf_kept(a.vocab, C, W);
    const size_t largest = (size_t)di.max_smem_optin - kVfStatic;
    const bool keep = !a.greedy && stats + kept <= largest;
    const size_t smem = stats + (keep ? kept : 0);
    const int mode = a.greedy ? VF_GREEDY : keep ? VF_KEEP : VF_AGAIN;
    auto k = a.greedy ? verify_kernel<C, W, VF_GREEDY> : keep ? verify_kernel<C, W, VF_KEEP> : verify_kernel<C, W, VF_AGAIN>;
    // The limit is the kernel's on this device, not the call's: set once, to the largest, so that
    // no call lowers it between another thread's setting and its launch.
    static std::atomic<uint64_t> ready[3];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("gbx_verify_tokens: device");
    if (!(ready[mode].load(std::memory_order_acquire) >> dev & 1)) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)largest) != cudaSuccess ||
            (C > 8 && cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
            return check_launch("gbx_verify_tokens: launch attributes");
        ready[mode].fetch_or((uint64_t)1 << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (pdl_enabled()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaLaunchKernelEx(&cfg, k, a);
    return check_launch("gbx_verify_tokens");
}

}  // namespace gbx

using namespace gbx;

extern "C" int gbx_verify_tokens(const float* logits, const float* draft_logits, const int32_t* draft_ids,
                                 const int32_t* draft_len, int64_t B, int n_draft, int vocab, double temperature,
                                 const double* uniforms, int32_t* out_ids, int32_t* n_accepted, int* err_flag,
                                 gbx_stream_t stream)
{
    if (B < 0 || n_draft < 0 || vocab <= 0)
        return set_error(GBX_EINVAL, "gbx_verify_tokens: B=%lld n_draft=%d vocab=%d", (long long)B, n_draft, vocab);
    // its reciprocal has to be an fp32 number
    if (!(temperature < 1e38)) return set_error(GBX_EINVAL, "gbx_verify_tokens: temperature %g", temperature);
    if (n_draft > kVfMaxDraft) return set_error(GBX_ERANGE, "gbx_verify_tokens: n_draft=%d (at most %d)", n_draft, kVfMaxDraft);
    if (B > 0x7fffffffLL / 16) return set_error(GBX_ERANGE, "gbx_verify_tokens: B=%lld", (long long)B);
    if (B == 0) return GBX_OK;
    const bool greedy = temperature <= 0.01;
    if (!logits || !out_ids || !n_accepted || (n_draft > 0 && !draft_ids))
        return set_error(GBX_EINVAL, "gbx_verify_tokens: null pointer");
    if (!greedy && !uniforms) return set_error(GBX_EINVAL, "gbx_verify_tokens: temperature %g needs uniforms", temperature);
    VfArgs a;
    a.logits = logits;
    a.draft_logits = draft_logits;
    a.draft_ids = draft_ids;
    a.draft_len = draft_len;
    a.n = n_draft;
    a.vocab = vocab;
    a.inv_t = greedy ? 1.0 : 1.0 / temperature;
    a.c2 = (float)(1.4426950408889634 * a.inv_t);
    a.greedy = greedy ? 1 : 0;
    a.uniforms = uniforms;
    a.out_ids = out_ids;
    a.n_accepted = n_accepted;
    a.err = err_flag;
    // One sequence of 4 drafts, 16 and 64 of up to 7, vocabulary 50257: 16, 28 and 79 us with
    // clusters of 16 CTAs of 8 warps, 19, 41 and 69 with 8 of 16, 26, 41 and 85 with 4 of 16.
    DeviceInfo di;
    if (device_info(&di) != GBX_OK) return GBX_ECUDA;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return B * 16 <= 2 * di.sm_count ? vf_launch<16, 8>(a, B, di, s) : vf_launch<8, 16>(a, B, di, s);
}
