// verify.cu -- verification of drafted tokens against the target's
// distributions (gbx_verify_tokens), beside the next-token selection of
// select.cu.  No counterpart in the reference (its generate loop takes one
// token per forward, transformer.cu:986-1036).
//
// One cluster of 4 to 16 CTAs per sequence, one launch; each of its warps owns
// one run of the vocabulary.
//   A  the rows' statistics: the warp's run of every target and draft row,
//      through a ring of four asynchronous copies; maximum and sum of
//      2^((x - m) log2(e) / T) in one pass (running maximum per lane).  fp32:
//      the sum decides a test whose border is a single point.
//   B  every CTA takes the same decision from the statistics and the drafted
//      tokens' own logits: the first draft that is not accepted.
//   C  the next token by inversion of the running sum of r_j = max(p_j - q_j,
//      0) (p_j after the last draft): the two normalisers, the runs' sums, and
//      then the one run that holds the border.  A lane owns 16 neighbouring
//      entries, so a run's sum, its lanes' prefixes and the entry are found
//      from the same 16 registers.  fp64: a vocabulary has a border every few
//      1e-5 of the sum, so an error of 1e-7 in the running sum would pick a
//      neighbour every few hundred draws.
// What the CTAs tell one another they write into each other's shared memory
// before a cluster barrier, so that every read after it is local.
// At temperature <= 0.01 A finds each target row's first maximum and C is not
// needed.
//
// The fp64 exponential is table-driven (P. T. P. Tang, "Table-driven
// implementation of the exponential function in IEEE floating-point
// arithmetic", 1989): with t = 128 (x - m) / (T ln 2), one FMA of the logit,
// k = rint(t) and r = t - k, e^((x - m) / T) = 2^(k/128) e^(r ln 2 / 128), the
// second factor by its Taylor polynomial of degree 4 (|r ln 2 / 128| < 0.0028:
// remainder below 1.3e-15), the 128 roots computed into shared memory by
// exp2(): nine fp64 instructions where the fp64 pipe is what bounds C.
#include "gbx_common.cuh"
#include "kv_cache.cuh"

namespace gbx {

constexpr int kVfWarps = 8;
constexpr int kVfThreads = 32 * kVfWarps;
constexpr int kVfChunk = 512;    // entries a warp handles at a time
constexpr int kVfSlots = 4;      // chunks in flight
constexpr int kVfPad = kVfChunk + kVfChunk / 16;   // a chunk with one float of padding after every 16
constexpr int kVfMaxDraft = 256;
// dynamic shared memory: the ring (later the padded chunks), then the rows' statistics
constexpr size_t kVfRing = sizeof(float) * kVfWarps * kVfSlots * kVfChunk;
constexpr size_t vf_smem(int n, int cluster) { return kVfRing + sizeof(float2) * (2 * n + 1) * (kVfWarps + cluster + 1); }
static_assert(2 * kVfPad <= kVfSlots * kVfChunk, "two padded chunks fit a warp's ring");

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
__device__ __forceinline__ float2 vf_merge(float2 a, float2 b, float c2)
{
    const float m = fmaxf(a.x, b.x), base = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * vf_exp2((a.x - base) * c2) + b.y * vf_exp2((b.x - base) * c2));
}

__device__ __forceinline__ float2 vf_better(float2 a, float2 b)
{
    if (a.x != a.x) return a;
    if (b.x != b.x) return b;
    return b.x > a.x || (b.x == a.x && __float_as_int(b.y) < __float_as_int(a.y)) ? b : a;
}

// Of N neighbouring lanes' parts, in a fixed tree.
template <int N>
__device__ __forceinline__ float2 vf_reduce(float2 v, float c2, int greedy)
{
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const float2 w = make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
        v = greedy ? vf_better(v, w) : vf_merge(v, w, c2);
    }
    return v;
}

// The exponential of one distribution (see the header): e^((x - m) / T) of a
// logit x; 0 below e^-700.
struct VfExp {
    double c, d;          // t = x c + d
    const double* root;   // 2^(i/128)
    __device__ __forceinline__ VfExp(double m, double inv_t, const double* roots)
        : c(inv_t * 184.6649652337873), d(-m * (inv_t * 184.6649652337873)), root(roots)
    {
    }
    __device__ __forceinline__ double operator()(float x) const
    {
        const double t = fma((double)x, c, d);
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
template <int C>
__global__ void __launch_bounds__(kVfThreads, 2) verify_kernel(const VfArgs a)
{
    constexpr int kVfRuns = C * kVfWarps;
    grid_dependency_wait();
    vf_arrive();   // awaited before the first write into another CTA
    extern __shared__ __align__(16) float vf_smem_raw[];
    __shared__ double s_root[128];
    __shared__ double s_z[2][kVfRuns], s_run[kVfRuns];
    __shared__ int s_dec;         // accepted drafts
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int64_t b = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = a.n, V = a.vocab, max_rows = 2 * n + 1;
    float* ring = vf_smem_raw + warp * kVfSlots * kVfChunk;
    float2* s_warp = reinterpret_cast<float2*>(vf_smem_raw + kVfWarps * kVfSlots * kVfChunk);   // [rows][warps]
    float2* s_part = s_warp + max_rows * kVfWarps;                                              // [rows][CTAs]
    float2* s_stat = s_part + max_rows * C;                                            // [rows]
    int len = a.draft_len ? a.draft_len[b] : n;
    const bool bad_len = len < 0 || len > n;
    if (bad_len) len = 0;
    const float* tl = a.logits + b * (n + 1) * (int64_t)V;
    const float* dl = a.draft_logits && !a.greedy ? a.draft_logits + b * (int64_t)n * V : nullptr;
    const int32_t* ids = a.draft_ids + b * n;
    // this warp's run of every row, in chunks
    const int run = (V + kVfRuns - 1) / kVfRuns;
    const int me = (int)rank * kVfWarps + warp;
    const int j0 = min(V, me * run), j1 = min(V, j0 + run);
    const int chunks = (run + kVfChunk - 1) / kVfChunk;
    const int nrows = bad_len ? 0 : len + 1 + (dl ? len : 0);
    auto row = [&](int k) { return k <= len ? tl + (int64_t)k * V : dl + (int64_t)(k - len - 1) * V; };

    // ---------------------------------------------------- A
    // unit u: chunk u % chunks of row u / chunks
    auto fetch = [&](int k, int ch, int slot) {
        const float* x = row(k);
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + slot * kVfChunk + lane);
        const int j = j0 + ch * kVfChunk + lane;
#pragma unroll
        for (int e = 0; e < kVfChunk / 32; ++e)
            if (j + 32 * e < j1) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 128 * e), "l"(x + j + 32 * e) : "memory");
    };
    int fk = 0, fc = 0;   // the unit that is fetched next
    auto fetch_next = [&](int slot) {
        if (fk < nrows) fetch(fk, fc, slot);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++fc == chunks) {
            fc = 0;
            ++fk;
        }
    };
#pragma unroll
    for (int i = 0; i < kVfSlots - 1; ++i) fetch_next(i);
    // what B and C need from memory, asked for meanwhile
    const double u_next = a.greedy ? 0.0 : a.uniforms[b * (n + 1) + n];
    int d_mine = -1;
    float tl_mine = 0.0f, dl_mine = 0.0f;
    double u_mine = 0.0;
    if (tid < len) {
        d_mine = ids[tid];
        if (!a.greedy) u_mine = a.uniforms[b * (n + 1) + tid];
        if ((unsigned)d_mine < (unsigned)V) {
            tl_mine = tl[(int64_t)tid * V + d_mine];
            if (dl) dl_mine = dl[(int64_t)tid * V + d_mine];
        }
    }
    if (tid < 128) s_root[tid] = exp2(tid * (1.0 / 128.0));
    if (tid == 0) s_dec = len;
    int slot = 0;
#pragma unroll 2
    for (int k = 0; k < nrows; ++k) {
        float m = -INFINITY, s = 0.0f;
        int at = 0x7fffffff;
        bool nan = false;
        for (int ch = 0; ch < chunks; ++ch) {
            __syncwarp();   // every lane has read the slot that is filled next
            fetch_next(slot ? slot - 1 : kVfSlots - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kVfSlots - 1) : "memory");
            __syncwarp();
            float v[kVfChunk / 32];
            const int j = j0 + ch * kVfChunk + lane;
#pragma unroll
            for (int e = 0; e < kVfChunk / 32; ++e) v[e] = j + 32 * e < j1 ? ring[slot * kVfChunk + lane + 32 * e] : -INFINITY;
            if (a.greedy) {
#pragma unroll
                for (int e = 0; e < kVfChunk / 32; ++e) {
                    nan |= v[e] != v[e];
                    if (v[e] > m) {
                        m = v[e];
                        at = j + 32 * e;
                    }
                }
            } else {
                float bm = fmaxf(m, v[0]);
#pragma unroll
                for (int e = 1; e < kVfChunk / 32; ++e) bm = fmaxf(bm, v[e]);
                const float base = (bm == -INFINITY ? 0.0f : bm) * a.c2;
                float t = 0.0f, t1 = 0.0f;
#pragma unroll
                for (int e = 0; e < kVfChunk / 32; e += 2) {   // a NaN makes the sum NaN
                    t += vf_exp2(fmaf(v[e], a.c2, -base));
                    t1 += vf_exp2(fmaf(v[e + 1], a.c2, -base));
                }
                s = fmaf(s, vf_exp2(fmaf(m, a.c2, -base)), t + t1);   // m = -inf: 0
                m = bm;
            }
            slot = slot + 1 == kVfSlots ? 0 : slot + 1;
        }
        float2 st;
        if (a.greedy) {
            st = vf_reduce<32>(make_float2(nan ? __int_as_float(0x7fc00000) : m, __int_as_float(at)), a.c2, 1);
        } else {
            const float wm = group_max<32>(m), base = wm == -INFINITY ? 0.0f : wm;
            st = make_float2(wm, group_sum<32>(s * vf_exp2((m - base) * a.c2)));
        }
        if (lane == 0) s_warp[k * kVfWarps + warp] = st;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    vf_wait();   // the other CTAs run
    // this CTA's part of each row, to every CTA
    for (int i = tid; i < (nrows * kVfWarps + 31 & ~31); i += kVfThreads) {
        const int k = i / kVfWarps, w = i % kVfWarps;
        const float2 t = vf_reduce<kVfWarps>(k < nrows ? s_warp[i] : make_float2(-INFINITY, 0.0f), a.c2, a.greedy);
        if (k < nrows)
            for (uint32_t p = w; p < C; p += kVfWarps) vf_push(s_part + k * C + rank, p, t);
    }
    vf_arrive();
    vf_wait();
    // the whole rows; x NaN: the row gives no distribution
    for (int i = tid; i < (nrows * C + 31 & ~31); i += kVfThreads) {
        const int k = i / C;
        float2 t = vf_reduce<C>(k < nrows ? s_part[i] : make_float2(-INFINITY, 0.0f), a.c2, a.greedy);
        if (fabsf(t.x) == INFINITY || (!a.greedy && t.y != t.y)) t.x = __int_as_float(0x7fc00000);
        if (k < nrows && i % C == 0) s_stat[k] = t;
    }
    __syncthreads();

    // ---------------------------------------------------- B
    if (tid < len) {
        const float2 st = s_stat[tid];
        const bool known = (unsigned)d_mine < (unsigned)V;
        if (!known && rank == 0) kv_flag(a.err, GBX_VERIFY_BAD_ID);
        bool ok = st.x == st.x && known;
        if (ok && a.greedy) {
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
        const int next = a.greedy && !bad ? __float_as_int(sp.y) : -1;
        for (int i = tid; i <= n; i += kVfThreads)
            if (i != acc || a.greedy || bad) a.out_ids[b * (n + 1) + i] = i < acc ? ids[i] : i == acc ? next : -1;
        if (tid == 0) {
            a.n_accepted[b] = acc;
            if (bad) kv_flag(a.err, GBX_VERIFY_BAD_ROW);
        }
    }
    if (a.greedy || bad) return;   // every CTA of the cluster alike

    // ---------------------------------------------------- C
    const float* px = tl + (int64_t)acc * V;
    const float* qx = rejected && dl ? dl + (int64_t)acc * V : nullptr;
    const int hot = rejected && !dl ? ids[acc] : -1;   // a draft picked without chance
    const VfExp pexp(sp.x, a.inv_t, s_root), qexp(sq.x, a.inv_t, s_root);
    // e^((x - m) / T) of entries j0 + 512 ch + 16 lane + e: read coalesced, turned in shared memory
    double ep[16], eq[16];
    auto load = [&](int ch) {
        const int j = j0 + ch * kVfChunk + lane;
        float x[16], y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = j + 32 * e < j1 ? px[j + 32 * e] : -INFINITY;
        if (qx)
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = j + 32 * e < j1 ? qx[j + 32 * e] : -INFINITY;
        __syncwarp();
        float* turn = ring + lane + (lane >> 4);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            turn[34 * e] = x[e];
            if (qx) turn[kVfPad + 34 * e] = y[e];
        }
        __syncwarp();
        const float* mine = ring + 17 * lane;
#pragma unroll
        for (int e = 0; e < 16; ++e) ep[e] = pexp(mine[e]);
#pragma unroll
        for (int e = 0; e < 16; ++e) eq[e] = qx ? qexp(mine[kVfPad + e]) : 0.0;
    };
    auto sum32 = [](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    double zp = 0.0, zq = 0.0;
    for (int ch = 0; ch < chunks; ++ch) {
        load(ch);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            zp += ep[e];
            zq += eq[e];
        }
    }
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
    // entry e's weight of the chunk that is loaded
    auto weight = [&](int ch, int e) {
        // rounded products: equal p and q leave exactly nothing, and every evaluation the same
        const double p = __dmul_rn(ep[e], ip);
        if (!minus) return p;
        const double q = qx ? __dmul_rn(eq[e], iq) : j0 + ch * kVfChunk + 16 * lane + e == hot ? 1.0 : 0.0;
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
        double t = 0.0;
        for (int ch = 0; ch < chunks; ++ch) {
            if (chunks > 1) load(ch);
#pragma unroll
            for (int e = 0; e < 16; ++e) t += weight(ch, e);
        }
        t = sum32(t);
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
        double cum = __shfl_sync(0xffffffffu, at_run, owner);
        if (found != me) return;
        int pick = -1, last = -1;   // last: the run's last entry with any weight, should rounding end the run early
        for (int ch = 0; ch < chunks && pick < 0; ++ch) {
            if (chunks > 1) load(ch);
            double w[16], sum = 0.0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                w[e] = weight(ch, e);
                sum += w[e];
            }
            const double c = scan32(sum);
            double at = cum + (c - sum);
            int first = 0x7fffffff, tail = -1;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                at += w[e];
                if (w[e] > 0.0) {
                    tail = e;
                    if (at > want) first = min(first, e);
                }
            }
            const int j = j0 + ch * kVfChunk + 16 * lane;
            first = __reduce_min_sync(0xffffffffu, first == 0x7fffffff ? first : j + first);
            last = max(last, __reduce_max_sync(0xffffffffu, tail < 0 ? -1 : j + tail));
            if (first != 0x7fffffff) pick = first;
            cum += __shfl_sync(0xffffffffu, c, 31);
        }
        if (lane == 0) a.out_ids[b * (n + 1) + acc] = pick >= 0 ? pick : last;
        return;
    }
}

template <int C>
static int vf_launch(const VfArgs& a, int64_t B, cudaStream_t s)
{
    auto k = verify_kernel<C>;
    const size_t smem = vf_smem(a.n, C);
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        (C > 8 && cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
        return check_launch("gbx_verify_tokens: launch attributes");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(kVfThreads);
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
    if (!(temperature < INFINITY)) return set_error(GBX_EINVAL, "gbx_verify_tokens: temperature %g", temperature);
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
    // CTAs per sequence: the fewer, the less is spent on meeting; 16 while every
    // sequence's cluster then still runs at once (two CTAs to an SM), else 8, else 4
    DeviceInfo di;
    if (device_info(&di) != GBX_OK) return GBX_ECUDA;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#ifdef VFC
    return vf_launch<VFC>(a, B, s);
#endif
    if (B * 16 <= 2 * di.sm_count) return vf_launch<16>(a, B, s);
    if (B * 8 <= 2 * di.sm_count) return vf_launch<8>(a, B, s);
    return vf_launch<4>(a, B, s);
}
