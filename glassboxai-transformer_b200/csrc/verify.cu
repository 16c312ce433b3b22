// verify.cu -- verification of drafted tokens against the target's
// distributions (gbx_verify_tokens), beside the next-token selection of
// select.cu.  No counterpart in the reference (its generate loop takes one
// token per forward, transformer.cu:986-1036).
//
// One cluster of 8 CTAs per sequence, one launch:
//   A  the rows' statistics: row k of the sequence's target and draft rows
//      goes to CTA k mod 8; maximum and sum of 2^((x - m) log2(e) / T) in one
//      pass (running maximum per thread).  fp32: the sum decides a test whose
//      border is a single point.
//   B  every CTA takes the same decision from the statistics and the drafted
//      tokens' own logits: the first draft that is not accepted.
//   C  the next token by inversion of the running sum of r_j = max(p_j - q_j,
//      0) (p_j after the last draft), over 128 warps, each with one run of
//      the vocabulary: the two normalisers, the runs' sums, and then the one
//      run that holds the border, 32 entries at a time.  fp64: a vocabulary has
//      a border every few 1e-5 of the sum, so an error of 1e-7 in the running
//      sum would pick a neighbour every few hundred draws.
// At temperature <= 0.01 A finds each target row's first maximum and C is not
// needed.
//
// The fp64 exponential is table-driven (P. T. P. Tang, "Table-driven
// implementation of the exponential function in IEEE floating-point
// arithmetic", 1989): e^y = 2^(k/64) e^r, k = round(64 y / ln 2), |r| <= ln 2
// / 128, with e^r by its Taylor polynomial of degree 5 (remainder r^6 / 720 <
// 4e-17) and the 64 roots computed into shared memory by exp2(): about 11 fp64
// instructions where the fp64 pipe is what bounds C.
#include "gbx_common.cuh"
#include "kv_cache.cuh"

namespace gbx {

constexpr int kVfCluster = 8;
constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfRuns = kVfCluster * kVfWarps;
constexpr int kVfMaxDraft = 1024;
constexpr int kVfStats = (2 * kVfMaxDraft + 1 + kVfCluster - 1) / kVfCluster;

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

// A row's statistics: maximum (NaN: the row gives no distribution) and sum;
// greedy: maximum and its first index.
struct VfStat {
    float m;
    float s;   // greedy: the index, as int bits
};

__device__ __forceinline__ void vf_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ uint32_t vf_peer(const void* p, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}

__device__ __forceinline__ float vf_peer_f32(const float* p, uint32_t rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(vf_peer(p, rank)) : "memory");
    return v;
}

__device__ __forceinline__ double vf_peer_f64(const double* p, uint32_t rank)
{
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(vf_peer(p, rank)) : "memory");
    return v;
}

// Calls f(j, x[j]) for this thread's share of a row that may start at any
// 4-byte address: vectors of four between a ragged head and tail.
template <class F>
__device__ __forceinline__ void vf_row(const float* x, int V, F f)
{
    const int head = min(V, (int)((4 - (((uintptr_t)x >> 2) & 3)) & 3));
    const int quads = (V - head) >> 2;
    if ((int)threadIdx.x < head) f(threadIdx.x, x[threadIdx.x]);
    const float4* v = reinterpret_cast<const float4*>(x + head);
#pragma unroll 4
    for (int q = threadIdx.x; q < quads; q += kVfThreads) {
        const float4 t = v[q];
        const int j = head + 4 * q;
        f(j, t.x);
        f(j + 1, t.y);
        f(j + 2, t.z);
        f(j + 3, t.w);
    }
    const int j = head + 4 * quads + threadIdx.x;
    if (j < V) f(j, x[j]);
}

__device__ VfStat vf_stats(const float* x, int V, float c2, float* red_m, float* red_s)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY, s = 0.0f;
    bool bad = false;
    vf_row(x, V, [&](int, float v) {
        bad |= !(v < INFINITY);   // NaN or +inf
        if (v > m) {
            s *= vf_exp2((m - v) * c2);   // m = -inf: 0
            m = v;
        }
        // v = m = -inf would give NaN: such an entry adds nothing
        s += v == -INFINITY ? 0.0f : vf_exp2((v - m) * c2);
    });
    if (bad) m = INFINITY;
    const float wm = group_max<32>(m);
    s = m == -INFINITY ? 0.0f : s * vf_exp2((m - wm) * c2);
    s = group_sum<32>(s);
    if (lane == 0) {
        red_m[warp] = wm;
        red_s[warp] = s;
    }
    __syncthreads();
    float bm = red_m[0], bs = 0.0f;
    for (int w = 1; w < kVfWarps; ++w) bm = fmaxf(bm, red_m[w]);
    for (int w = 0; w < kVfWarps; ++w) bs += red_m[w] == -INFINITY ? 0.0f : red_s[w] * vf_exp2((red_m[w] - bm) * c2);
    __syncthreads();
    VfStat r;
    r.m = fabsf(bm) == INFINITY ? __int_as_float(0x7fc00000) : bm;
    r.s = bs;
    return r;
}

__device__ VfStat vf_argmax(const float* x, int V, float* red_m, float* red_s)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY;
    int at = 0x7fffffff;
    bool bad = false;
    vf_row(x, V, [&](int j, float v) {
        bad |= !(v < INFINITY);
        // a thread meets its entries in rising order but for the ragged head
        if (v > m || (v == m && j < at)) {
            m = v;
            at = j;
        }
    });
    if (bad) m = INFINITY;
    auto take = [&](float om, int oa) {
        if (om > m || (om == m && oa < at)) {
            m = om;
            at = oa;
        }
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        take(om, oa);
    }
    if (lane == 0) {
        red_m[warp] = m;
        red_s[warp] = __int_as_float(at);
    }
    __syncthreads();
    m = red_m[0];
    at = __float_as_int(red_s[0]);
    for (int w = 1; w < kVfWarps; ++w) take(red_m[w], __float_as_int(red_s[w]));
    __syncthreads();
    VfStat r;
    r.m = fabsf(m) == INFINITY ? __int_as_float(0x7fc00000) : m;
    r.s = __int_as_float(at);
    return r;
}

// e^y for y <= 0 (see the header); 0 below -700.
__device__ __forceinline__ double vf_exp(double y, const double* root)
{
    if (!(y > -700.0)) return 0.0;
    const double k = rint(y * 92.33248261689366);                  // 64 / ln 2
    double r = fma(k, -0.010830424696249145, y);                    // ln 2 / 64, rounded
    r = fma(k, -3.6235106466348431e-19, r);                                  // what the rounding left out
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(r, p, 1.0 / 6.0);
    p = fma(r, p, 0.5);
    p = fma(r, p, 1.0);
    p = fma(r, p, 1.0);
    const int ki = (int)k;
    const double t = root[ki & 63];
    return p * __hiloint2double(__double2hiint(t) + ((ki >> 6) << 20), __double2loint(t));   // exponent stays normal above -700
}

__global__ void __cluster_dims__(kVfCluster, 1, 1) __launch_bounds__(kVfThreads) verify_kernel(const VfArgs a)
{
    grid_dependency_wait();
    __shared__ float s_m[kVfStats], s_s[kVfStats];   // this CTA's rows
    __shared__ float red_m[kVfWarps], red_s[kVfWarps];
    __shared__ double s_root[64];
    __shared__ double s_z[2][kVfWarps], s_run[kVfWarps];
    __shared__ int s_dec;         // accepted drafts
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int64_t b = blockIdx.x / kVfCluster;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = a.n, V = a.vocab;
    int len = a.draft_len ? a.draft_len[b] : n;
    const bool bad_len = len < 0 || len > n;
    if (bad_len) len = 0;
    const float* tl = a.logits + b * (n + 1) * (int64_t)V;
    const float* dl = a.draft_logits && !a.greedy ? a.draft_logits + b * (int64_t)n * V : nullptr;
    const int32_t* ids = a.draft_ids + b * n;
    if (tid < 64) s_root[tid] = exp2(tid * (1.0 / 64.0));
    if (tid == 0) s_dec = len;

    // ---------------------------------------------------- A
    const int nrows = bad_len ? 0 : len + 1 + (dl ? len : 0);
    for (int k = (int)rank; k < nrows; k += kVfCluster) {
        const float* x = k <= len ? tl + (int64_t)k * V : dl + (int64_t)(k - len - 1) * V;
        const VfStat st = a.greedy ? vf_argmax(x, V, red_m, red_s) : vf_stats(x, V, a.c2, red_m, red_s);
        if (tid == 0) {
            s_m[k / kVfCluster] = st.m;
            s_s[k / kVfCluster] = st.s;
        }
    }
    vf_cluster_sync();
    auto stat = [&](int k) {
        VfStat r;
        r.m = vf_peer_f32(s_m + k / kVfCluster, k % kVfCluster);
        r.s = vf_peer_f32(s_s + k / kVfCluster, k % kVfCluster);
        return r;
    };

    // ---------------------------------------------------- B
    for (int i = tid; i < len; i += kVfThreads) {
        const VfStat st = stat(i);
        const int d = ids[i];
        const bool known = (unsigned)d < (unsigned)V;
        if (!known && rank == 0) kv_flag(a.err, GBX_VERIFY_BAD_ID);
        bool ok = st.m == st.m && known;
        if (ok && a.greedy) {
            ok = d == __float_as_int(st.s);
        } else if (ok) {
            double q = 1.0;
            if (dl) {
                const VfStat sq = stat(len + 1 + i);
                if (sq.m == sq.m) q = vf_exp(((double)dl[(int64_t)i * V + d] - (double)sq.m) * a.inv_t, s_root) / (double)sq.s;
                else ok = false;
            }
            const double p = vf_exp(((double)tl[(int64_t)i * V + d] - (double)st.m) * a.inv_t, s_root) / (double)st.s;
            ok = ok && a.uniforms[b * (n + 1) + i] * q < p;
        }
        if (!ok) atomicMin(&s_dec, i);
    }
    __syncthreads();
    const int acc = s_dec;
    const bool rejected = acc < len;
    bool bad = bad_len;
    VfStat sp{}, sq{};
    if (!bad) {
        sp = stat(acc);
        bad = !(sp.m == sp.m);
        if (rejected && dl) {
            sq = stat(len + 1 + acc);
            bad |= !(sq.m == sq.m);
        }
    }
    int next = -1;
    if (a.greedy && !bad) next = __float_as_int(sp.s);
    if (!a.greedy && !bad) {
        // ------------------------------------------------ C
        const float* px = tl + (int64_t)acc * V;
        const float* qx = rejected && dl ? dl + (int64_t)acc * V : nullptr;
        const int hot = rejected && !dl ? ids[acc] : -1;   // a draft picked without chance
        const int run = (V + kVfRuns - 1) / kVfRuns;
        const int me = (int)rank * kVfWarps + warp;
        const int j0 = min(V, me * run), j1 = min(V, j0 + run);
        const double pm = sp.m, qm = sq.m;
        double zp = 0.0, zq = 0.0;
        for (int j = j0 + lane; j < j1; j += 32) {
            zp += vf_exp(((double)px[j] - pm) * a.inv_t, s_root);
            if (qx) zq += vf_exp(((double)qx[j] - qm) * a.inv_t, s_root);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            zp += __shfl_xor_sync(0xffffffffu, zp, o);
            zq += __shfl_xor_sync(0xffffffffu, zq, o);
        }
        if (lane == 0) {
            s_z[0][warp] = zp;
            s_z[1][warp] = zq;
        }
        vf_cluster_sync();
        // every warp adds the 128 runs' sums in the same order
        auto total = [&](const double* mine) {
            double t = 0.0;
#pragma unroll
            for (int e = 0; e < kVfRuns / 32; ++e) {
                const int w = e * 32 + lane;
                t += vf_peer_f64(mine + w % kVfWarps, w / kVfWarps);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            return t;
        };
        const double ip = 1.0 / total(s_z[0]), iq = qx ? 1.0 / total(s_z[1]) : 0.0;
        bool minus = rejected;
        auto weight = [&](int j) {
            const double p = vf_exp(((double)px[j] - pm) * a.inv_t, s_root) * ip;
            if (!minus) return p;
            const double q = qx ? vf_exp(((double)qx[j] - qm) * a.inv_t, s_root) * iq : (j == hot ? 1.0 : 0.0);
            return fmax(p - q, 0.0);
        };
        for (int pass = 0; pass < 2; ++pass) {
            double t = 0.0;
            for (int j = j0 + lane; j < j1; j += 32) t += weight(j);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) s_run[warp] = t;
            vf_cluster_sync();
            // the running sum over the runs: lane l holds runs 4l .. 4l + 3
            double r[4], mine = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int w = lane * 4 + e;
                r[e] = vf_peer_f64(s_run + w % kVfWarps, w / kVfWarps);
                mine += r[e];
            }
            double incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            const double all = __shfl_sync(0xffffffffu, incl, 31);
            if (!(all > 0.0) && minus) {   // p = q: of p itself (every CTA alike)
                minus = false;
                vf_cluster_sync();         // the runs' sums have been read
                continue;
            }
            const double u = a.uniforms[b * (n + 1) + n];
            const double want = (u > 0.0 ? u : 0.0) * all;
            // the first run whose running sum passes `want`, and the sum before it
            int found = 0x7fffffff, any = -1;
            double before = incl - mine, at_run = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (found == 0x7fffffff && before + r[e] > want && r[e] > 0.0) {
                    found = lane * 4 + e;
                    at_run = before;
                }
                before += r[e];
                if (r[e] > 0.0) any = lane * 4 + e;
            }
            const unsigned who = __ballot_sync(0xffffffffu, found != 0x7fffffff);
            const unsigned some_run = __ballot_sync(0xffffffffu, any >= 0);
            // none (u * all rounded up to all): the last entry with any weight
            const int owner = who ? __ffs(who) - 1 : 31 - __clz(some_run);
            found = __shfl_sync(0xffffffffu, who ? found : any, owner);
            double cum = __shfl_sync(0xffffffffu, at_run, owner);
            if (found == me) {
                int pick = -1, last = -1;   // last: the run's last entry with any weight, should rounding end the run early
                for (int j = j0; j < j1 && pick < 0; j += 32) {
                    const double wgt = j + lane < j1 ? weight(j + lane) : 0.0;
                    double c = wgt;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double up = __shfl_up_sync(0xffffffffu, c, o);
                        if (lane >= o) c += up;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, cum + c > want && wgt > 0.0);
                    const unsigned some = __ballot_sync(0xffffffffu, wgt > 0.0);
                    if (over) pick = j + __ffs(over) - 1;
                    if (some) last = j + 31 - __clz(some);
                    cum += __shfl_sync(0xffffffffu, c, 31);
                }
                next = pick >= 0 ? pick : last;
                if (lane == 0) a.out_ids[b * (n + 1) + acc] = next;
            }
            break;
        }
        if (rank == 0) {
            for (int i = tid; i <= n; i += kVfThreads)
                if (i != acc) a.out_ids[b * (n + 1) + i] = i < acc ? ids[i] : -1;
            if (tid == 0) a.n_accepted[b] = acc;
        }
    } else if (rank == 0) {
        for (int i = tid; i <= n; i += kVfThreads) a.out_ids[b * (n + 1) + i] = i < acc ? ids[i] : i == acc ? next : -1;
        if (tid == 0) {
            a.n_accepted[b] = acc;
            if (bad) kv_flag(a.err, GBX_VERIFY_BAD_ROW);
        }
    }
    vf_cluster_sync();   // no CTA leaves while another may still read its shared memory
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
    if (B > 0x7fffffffLL / kVfCluster) return set_error(GBX_ERANGE, "gbx_verify_tokens: B=%lld", (long long)B);
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
    launch_row_kernel(verify_kernel, dim3((unsigned)(B * kVfCluster)), dim3(kVfThreads), 0,
                      reinterpret_cast<cudaStream_t>(stream), a);
    return check_launch("gbx_verify_tokens");
}
