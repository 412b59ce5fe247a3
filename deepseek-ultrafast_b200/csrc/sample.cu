// Token sampling from logits (dsuf_sample): temperature, top-k, top-p, min-p and one given uniform number per row.
//
// With M the largest logit of a row, weights w_i = exp((l_i - M) / T) and the order "larger logit first, lower id first among equals":
//   A = the first top_k tokens; B = those of A whose preceding weight inside A is below top_p * weight(A) (the first always);
//   C = those of B with w_i >= min_p (the first always); the drawn token is the lowest id i of C with weight(C, ids <= i) > u weight(C).
// The reference's sampler (crates/kernels/cu/sample.cu) merges the output head's records; this one works on the logits themselves, so that
// top_k and top_p have no limit.
//
// Nothing is sorted.  A cluster of up to 8 CTAs shares a row (latency-bound at few rows; the row comes from HBM once and from L2 in the
// later passes).  Weights are 40-bit fixed point, their sums 64-bit integers: exact, so the result depends neither on the split nor
// on the order of the histogram's atomics.  Passes:
//   1. largest and smallest logit
//   2. weights: their sum and, when top-k or top-p is on, counts and weights of 1024 bins of l (linear from M down, so that bins
//      are evenly filled; a monotone map, so bins are an order)
//   3. per limit, the tokens of the one bin where it falls are listed (usually some dozens) and ranked against each other: the limit becomes
//      a threshold (logit, id).  A bin with more than 512 tokens is split again by the bits of the logits, down to equal
//      ones, of which the id decides.
//   4. weight of C per warp, and the owner of the drawn number walks its part.
// The exponent is formed in 64 bits ((l - M) / T rounded to fp32 would be off by 1e-6 relative in a far token's weight).
#include "internal.h"

namespace dsuf {

constexpr int SA_THREADS = 512;
constexpr int SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = 1024;
constexpr int SA_LIST = 512;
constexpr int SA_MAX_CLUSTER = 8;
constexpr float SA_ONE = 1099511627776.f;   // weight 1 in fixed point: 2^40
typedef unsigned long long u64;

struct SampleArgs {
    const float* logits;
    long long ld;
    int n;
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* ids;
    float* logprobs;
};

// The same shared-memory object of CTA `rank` of the cluster.
template <typename T>
DSUF_DEV T* in_cta(T* p, uint32_t rank) {
    u64 a = (u64)p, r;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(a), "r"(rank));
    return (T*)r;
}

DSUF_DEV uint32_t order_key(float l) {   // unsigned that orders like the float
    const uint32_t b = __float_as_uint(l);
    return (b >> 31) ? ~b : (b | 0x80000000u);
}
DSUF_DEV float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }

struct SampleShared {
    uint32_t count[SA_BINS];         // this CTA's histogram
    u64 mass[SA_BINS];
    uint32_t all_count[SA_BINS];     // the row's
    u64 all_mass[SA_BINS];
    uint32_t list_key[SA_LIST];      // this CTA's tokens of the limit's bin
    int list_id[SA_LIST];
    uint32_t row_key[SA_LIST];       // the row's
    int row_id[SA_LIST];
    u64 row_w[SA_LIST];
    uint32_t n_list;
    float top[SA_MAX_CLUSTER], low[SA_MAX_CLUSTER], lp[SA_MAX_CLUSTER];
    int first[SA_MAX_CLUSTER];
    u64 kept[SA_MAX_CLUSTER];
    uint32_t key_hi[SA_MAX_CLUSTER], key_lo[SA_MAX_CLUSTER], ties[SA_MAX_CLUSTER];
    u64 warp_a[SA_WARPS];
    uint32_t warp_b[SA_WARPS];
    float warp_f[SA_WARPS], warp_g[SA_WARPS];
    int found_bin;
    u64 found_mass, found_a, found_b;
    uint32_t found_count, found_key;
    int found_id;
};

struct Sampler {
    const SampleArgs& a;
    SampleShared& s;
    const float* x;          // the row
    int lead;                // elements between the 16-byte line of x[0] and x[0]
    int v0, v1;              // this warp's 16-byte lines
    int tid, warp, lane;
    uint32_t rank, ctas;
    float top, inv_bin;
    double inv_temp;
    bool stale;              // the row's histogram has been replaced by a split bin's

    DSUF_DEV float clean(float l) const { return l == l ? l + 0.f : -INFINITY; }   // NaN is never drawn; -0 orders as 0
    DSUF_DEV void line(int v, float* l) const {
        const int i = 4 * v - lead;
        if (i >= 0 && i + 4 <= a.n) {
            const float4 q = *reinterpret_cast<const float4*>(x + i);
            l[0] = clean(q.x); l[1] = clean(q.y); l[2] = clean(q.z); l[3] = clean(q.w);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) l[e] = i + e >= 0 && i + e < a.n ? clean(x[i + e]) : -INFINITY;
        }
    }
    // f(id, logit) for every element of this warp's part (ids outside the row come as -inf)
    template <typename F>
    DSUF_DEV void each(F f) const {
        int v = v0 + lane;
        for (; v + 96 < v1; v += 128) {     // four lines in flight
            float l[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) line(v + 32 * j, l[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) f(4 * (v + 32 * j) - lead + e, l[j][e]);
        }
        for (; v < v1; v += 32) {
            float l[4];
            line(v, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) f(4 * v - lead + e, l[e]);
        }
    }
    DSUF_DEV float weight(float l) const {
        if (l == top) return 1.f;
        const double z = ((double)l - (double)top) * inv_temp;
        const float hi = (float)z;
        if (!(hi > -80.f)) return 0.f;
        return expf(hi) * (1.f + (float)(z - (double)hi));
    }
    DSUF_DEV u64 fixed(float w) const { return (u64)(w * SA_ONE); }
    DSUF_DEV int bin(float l) const {
        if (l == top) return 0;
        const float f = (top - l) * inv_bin;
        return f < (float)(SA_BINS - 1) ? (int)f : SA_BINS - 1;
    }
    // f(sum, value) over the CTA; the result in every thread
    DSUF_DEV u64 block_sum(u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) s.warp_a[warp] = v;
        __syncthreads();
        u64 r = 0;
#pragma unroll
        for (int w = 0; w < SA_WARPS; ++w) r += s.warp_a[w];
        return r;
    }

    // ---- a limit: by count (top-k: `want` tokens) or by weight (top-p: the token whose weight reaches `target`) ----
    struct Limit {
        uint32_t key;     // the last token inside: everything of a larger key, and of this key the ids up to `id`
        int id;
        u64 mass;         // weight of all inside
    };
    DSUF_DEV static bool inside(const Limit& lim, uint32_t key, int id) { return key > lim.key || (key == lim.key && id <= lim.id); }

    DSUF_DEV void clear_bins() {
        for (int i = tid; i < SA_BINS; i += SA_THREADS) {
            s.count[i] = 0;
            s.mass[i] = 0;
        }
        __syncthreads();
    }
    // the CTAs' histograms into everybody's all_count / all_mass
    DSUF_DEV void share_bins() {
        cluster_barrier();
        const int per = SA_BINS / ctas;
        for (int i = tid; i < per; i += SA_THREADS) {
            const int b = rank * per + i;
            uint32_t c = 0;
            u64 m = 0;
            for (uint32_t r = 0; r < ctas; ++r) {
                c += *in_cta(&s.count[b], r);
                m += *in_cta(&s.mass[b], r);
            }
            for (uint32_t r = 0; r < ctas; ++r) {
                *in_cta(&s.all_count[b], r) = c;
                *in_cta(&s.all_mass[b], r) = m;
            }
        }
        cluster_barrier();
    }
    // first bin where count (or weight) reaches the limit, counting from `count0` / `mass0`: bin, and what lies before it
    DSUF_DEV void find_bin(bool by_mass, u64 want, double target, u64 count0, u64 mass0, int only_bin, u64 only_mass) {
        constexpr int PER = SA_BINS / SA_THREADS;
        uint32_t c[PER];
        u64 m[PER], cs = 0, ms = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int b = tid * PER + e;
            c[e] = s.all_count[b];
            m[e] = b == only_bin ? only_mass : b > only_bin ? 0 : s.all_mass[b];   // (top-p inside A: A's last bin counts with its part)
            cs += c[e];
            ms += m[e];
        }
        u64 ci = cs, mi = ms;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 cv = __shfl_up_sync(0xffffffffu, ci, o), mv = __shfl_up_sync(0xffffffffu, mi, o);
            if (lane >= o) { ci += cv; mi += mv; }
        }
        __syncthreads();
        if (lane == 31) {
            s.warp_a[warp] = mi;
            s.warp_b[warp] = (uint32_t)ci;
        }
        if (tid == 0) s.found_bin = -1;
        __syncthreads();
        u64 cb = count0 + ci - cs, mb = mass0 + mi - ms;
        for (int w = 0; w < warp; ++w) { cb += s.warp_b[w]; mb += s.warp_a[w]; }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const bool hit = by_mass ? (double)mb < target && target <= (double)(mb + m[e]) : cb < want && want <= cb + c[e];
            if (hit) {
                s.found_bin = tid * PER + e;
                s.found_a = cb;
                s.found_mass = mb;
                s.found_count = c[e];
            }
            cb += c[e];
            mb += m[e];
        }
        __syncthreads();
    }

    // The limit inside the row's histogram (all_count / all_mass of bin()).  `within`: only tokens inside this earlier limit count
    // (top-p inside A), or null.
    DSUF_DEV Limit limit(bool by_mass, u64 want, double target, const Limit* within) {
        int only_bin = SA_BINS;
        u64 only_mass = 0;
        if (within) {
            only_bin = bin(key_value(within->key));
            u64 before = 0;
            for (int i = tid; i < only_bin; i += SA_THREADS) before += s.all_mass[i];
            only_mass = within->mass - block_sum(before);
        }
        find_bin(by_mass, want, target, 0, 0, only_bin, only_mass);
        const int b0 = s.found_bin;
        u64 count0 = s.found_a, mass0 = s.found_mass;
        uint32_t n_in = s.found_count, k_hi = 0xffffffffu, k_lo = 0;
        __syncthreads();
        auto mine = [&](int id, float l) {
            if (l == -INFINITY || bin(l) != b0) return false;
            const uint32_t k = order_key(l);
            return k >= k_lo && k <= k_hi && (!within || inside(*within, k, id));
        };
        bool first_split = true;
        while (n_in > SA_LIST && k_hi != k_lo) {
            // split the bin by its logits' bits
            if (first_split) {
                uint32_t hi = 0, lo = 0xffffffffu;
                each([&](int id, float l) {
                    if (mine(id, l)) {
                        hi = max(hi, order_key(l));
                        lo = min(lo, order_key(l));
                    }
                });
                hi = __reduce_max_sync(0xffffffffu, hi);
                lo = __reduce_min_sync(0xffffffffu, lo);
                if (tid == 0) { s.key_hi[rank] = 0; s.key_lo[rank] = 0xffffffffu; }
                __syncthreads();
                if (lane == 0) { atomicMax(&s.key_hi[rank], hi); atomicMin(&s.key_lo[rank], lo); }
                cluster_barrier();
                k_hi = 0; k_lo = 0xffffffffu;
                for (uint32_t r = 0; r < ctas; ++r) {
                    k_hi = max(k_hi, *in_cta(&s.key_hi[r], r));
                    k_lo = min(k_lo, *in_cta(&s.key_lo[r], r));
                }
                first_split = false;
            }
            int shift = 0;
            while (((k_hi - k_lo) >> shift) >= (uint32_t)SA_BINS) ++shift;
            cluster_barrier();               // (the others are through with this CTA's histogram and keys)
            stale = true;
            clear_bins();
            each([&](int id, float l) {
                if (mine(id, l)) {
                    const uint32_t b = (k_hi - order_key(l)) >> shift;
                    atomicAdd(&s.count[b], 1u);
                    atomicAdd(&s.mass[b], fixed(weight(l)));
                }
            });
            share_bins();
            find_bin(by_mass, want, target, count0, mass0, SA_BINS, 0);
            const uint32_t b = (uint32_t)s.found_bin;
            count0 = s.found_a;
            mass0 = s.found_mass;
            n_in = s.found_count;
            __syncthreads();
            k_hi -= b << shift;
            k_lo = max(k_lo, k_hi - ((1u << shift) - 1u));
        }
        Limit out;
        if (n_in <= SA_LIST) {
            // list the tokens, everybody gets them all, every thread ranks one
            if (tid == 0) s.n_list = 0;
            __syncthreads();
            each([&](int id, float l) {
                if (mine(id, l)) {
                    const uint32_t at = atomicAdd(&s.n_list, 1u);
                    if (at < SA_LIST) {
                        s.list_key[at] = order_key(l);
                        s.list_id[at] = id;
                    }
                }
            });
            cluster_barrier();
            uint32_t base = 0;
            for (uint32_t r = 0; r < ctas; ++r) {
                const uint32_t n = min(*in_cta(&s.n_list, r), (uint32_t)SA_LIST);
                for (uint32_t i = tid; i < n && base + i < SA_LIST; i += SA_THREADS) {
                    const uint32_t k = *in_cta(&s.list_key[i], r);
                    s.row_key[base + i] = k;
                    s.row_id[base + i] = *in_cta(&s.list_id[i], r);
                    s.row_w[base + i] = fixed(weight(key_value(k)));
                }
                base = min(base + n, (uint32_t)SA_LIST);
            }
            cluster_barrier();               // (nobody reads this CTA's list any more)
            for (uint32_t i = tid; i < base; i += SA_THREADS) {
                const uint32_t k = s.row_key[i];
                const int id = s.row_id[i];
                u64 c = count0, m = mass0;
                for (uint32_t j = 0; j < base; ++j) {
                    const uint32_t kj = s.row_key[j];
                    if (kj > k || (kj == k && s.row_id[j] < id)) {
                        ++c;
                        m += s.row_w[j];
                    }
                }
                const u64 after = m + s.row_w[i];
                if (by_mass ? (double)m < target && target <= (double)after : c + 1 == want) {
                    s.found_key = k;
                    s.found_id = id;
                    s.found_b = after;
                }
            }
            __syncthreads();
            out.key = s.found_key;
            out.id = s.found_id;
            out.mass = s.found_b;
            __syncthreads();
            return out;
        }
        // many equal logits: the r-th lowest id among them
        const u64 w = fixed(weight(key_value(k_hi)));
        u64 r = by_mass ? (u64)ceil((target - (double)mass0) / (double)(w ? w : 1)) : want - count0;
        r = max(r, (u64)1);
        r = min(r, (u64)n_in);
        out.key = k_hi;
        out.mass = mass0 + r * w;
        uint32_t eq = 0;
        each([&](int id, float l) { eq += mine(id, l) ? 1u : 0u; });
        eq = __reduce_add_sync(0xffffffffu, eq);
        __syncthreads();
        if (lane == 0) s.warp_b[warp] = eq;
        __syncthreads();
        if (tid == 0) {
            uint32_t t = 0;
            for (int q = 0; q < SA_WARPS; ++q) t += s.warp_b[q];
            for (uint32_t q = 0; q < ctas; ++q) *in_cta(&s.ties[rank], q) = t;
        }
        cluster_barrier();
        u64 before = 0;
        for (uint32_t q = 0; q < rank; ++q) before += s.ties[q];
        for (int q = 0; q < warp; ++q) before += s.warp_b[q];
        if (before < r && r <= before + eq) {
            // this warp holds it: walk its lines in order
            for (int v = v0; v < v1; v += 32) {
                float l[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (v + lane < v1) line(v + lane, l);
                uint32_t c = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) c += mine(4 * (v + lane) - lead + e, l[e]) ? 1u : 0u;
                uint32_t upto = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                u64 at = before + upto - c;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (mine(4 * (v + lane) - lead + e, l[e]) && ++at == r)
                        for (uint32_t q = 0; q < ctas; ++q) *in_cta(&s.found_id, q) = 4 * (v + lane) - lead + e;
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        cluster_barrier();
        out.id = s.found_id;
        __syncthreads();
        return out;
    }
};

__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(const SampleArgs a) {
    __shared__ SampleShared s;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t rank = cluster_cta_rank(), ctas = cluster_num_ctas();
    const int row = blockIdx.x / ctas;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* x = a.logits + (size_t)row * a.ld;
    const int lead = (int)(((uintptr_t)x >> 2) & 3);
    const int lines = (int)(((long long)a.n + lead + 3) / 4);
    const long long parts = (long long)ctas * SA_WARPS, part = (long long)rank * SA_WARPS + warp;
    Sampler z{a, s, x, lead, (int)(lines * part / parts), (int)(lines * (part + 1) / parts), tid, warp, lane, rank, ctas, 0.f, 0.f, 0.0, false};
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;
    const bool greedy = !(temp > 0.f);

    // ---- pass 1: largest and smallest logit, and the first place of the largest ----
    float hi = -INFINITY, lo = INFINITY;
    int at = 0x7fffffff;
    z.each([&](int id, float l) {
        if (l > hi) { hi = l; at = id; }           // (a thread meets its ids in ascending order)
        if (l > -INFINITY) lo = fminf(lo, l);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float h = __shfl_xor_sync(0xffffffffu, hi, o);
        const int i = __shfl_xor_sync(0xffffffffu, at, o);
        if (h > hi || (h == hi && i < at)) { hi = h; at = i; }
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (lane == 0) { s.warp_f[warp] = hi; s.warp_g[warp] = lo; s.warp_b[warp] = (uint32_t)at; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SA_WARPS; ++w) {
            if (s.warp_f[w] > hi || (s.warp_f[w] == hi && (int)s.warp_b[w] < at)) { hi = s.warp_f[w]; at = (int)s.warp_b[w]; }
            lo = fminf(lo, s.warp_g[w]);
        }
        s.top[rank] = hi; s.low[rank] = lo; s.first[rank] = at;
    }
    cluster_barrier();
    hi = -INFINITY; lo = INFINITY; at = 0x7fffffff;
    for (uint32_t r = 0; r < ctas; ++r) {
        const float h = *in_cta(&s.top[r], r);
        const int i = *in_cta(&s.first[r], r);
        if (h > hi || (h == hi && i < at)) { hi = h; at = i; }
        lo = fminf(lo, *in_cta(&s.low[r], r));
    }
    z.top = hi;
    if (hi == -INFINITY) {    // nothing to draw from
        if (rank == 0 && tid == 0) {
            a.ids[row] = -1;
            if (a.logprobs) a.logprobs[row] = -INFINITY;
        }
        cluster_barrier();
        return;
    }
    z.inv_temp = greedy ? 1.0 : 1.0 / (double)temp;
    const float span = fminf(hi - lo, fmaxf(24.f, 32.f * temp));
    z.inv_bin = span > 0.f && span < INFINITY ? (float)(SA_BINS - 1) / span : 0.f;

    // ---- pass 2: weights; the log-probability's sum at temperature 1 ----
    const bool limited = !greedy && (top_k > 0 || top_p < 1.f);
    if (limited) z.clear_bins();
    u64 sum = 0;
    float lp = 0.f;
    uint32_t tokens = 0;
    if (!greedy || a.logprobs) {
        z.each([&](int id, float l) {
            if (l == -INFINITY) return;
            if (a.logprobs) lp += l == hi ? 1.f : expf(l - hi);
            if (greedy) return;
            const float w = z.weight(l);
            const u64 f = z.fixed(w);
            if (limited) {
                const int b = z.bin(l);
                ++tokens;
                sum += f;
                atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.mass[b], f);
            } else if (w >= min_p || l == hi) {
                sum += f;
            }
        });
    }
    if (a.logprobs) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lp += __shfl_xor_sync(0xffffffffu, lp, o);
        __syncthreads();
        if (lane == 0) s.warp_f[warp] = lp;
        __syncthreads();
        if (tid == 0) {
            float t = 0.f;
            for (int w = 0; w < SA_WARPS; ++w) t += s.warp_f[w];
            s.lp[rank] = t;
        }
    }
    Sampler::Limit lim;
    lim.key = order_key(-INFINITY) + 1;    // every token above -inf
    lim.id = 0x7fffffff;
    lim.mass = 0;
    if (limited) {
        // the row's number of tokens and weight
        const u64 n_mine = z.block_sum(tokens), m_mine = z.block_sum(sum);
        if (tid == 0) { s.kept[rank] = m_mine; s.ties[rank] = (uint32_t)n_mine; }
        z.share_bins();
        u64 n_all = 0, m_all = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
            n_all += *in_cta(&s.ties[r], r);
            m_all += *in_cta(&s.kept[r], r);
        }
        lim.mass = m_all;
        const bool cut = top_k > 0 && (u64)top_k < n_all;
        if (cut) lim = z.limit(false, (u64)top_k, 0.0, nullptr);
        if (top_p < 1.f) {
            // the first token is always inside: a target below one unit of weight is reached by it
            const double target = fmax((double)top_p * (double)lim.mass, 0.5);
            const Sampler::Limit k = lim;
            if (z.stale) {
                cluster_barrier();
                z.clear_bins();
                z.each([&](int id, float l) {
                    if (l == -INFINITY) return;
                    atomicAdd(&s.count[z.bin(l)], 1u);
                    atomicAdd(&s.mass[z.bin(l)], z.fixed(z.weight(l)));
                });
                z.share_bins();
            }
            lim = z.limit(true, 0, target, cut ? &k : nullptr);
        }
        sum = 0;
        z.each([&](int id, float l) {
            if (l > -INFINITY && Sampler::inside(lim, order_key(l), id)) {
                const float w = z.weight(l);
                if (w >= min_p || l == hi) sum += z.fixed(w);
            }
        });
    }

    // ---- the draw ----
    int token = at;
    if (!greedy) {
        u64 mine = sum;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        __syncthreads();
        if (lane == 0) s.warp_a[warp] = mine;
        __syncthreads();
        cluster_barrier();      // (kept is read no more as the row's weight)
        if (tid == 0) {
            u64 t = 0;
            for (int w = 0; w < SA_WARPS; ++w) t += s.warp_a[w];
            for (uint32_t r = 0; r < ctas; ++r) *in_cta(&s.kept[rank], r) = t;
        }
        cluster_barrier();
        u64 total = 0, before = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
            if (r < rank) before += s.kept[r];
            total += s.kept[r];
        }
        for (int w = 0; w < warp; ++w) before += s.warp_a[w];
        const float u = a.u[row];
        u64 draw = u > 0.f ? (u64)((double)u * (double)total) : 0;
        draw = min(draw, total - 1);
        if (before <= draw && draw < before + mine) {
            // this warp's part holds the token: walk it in the order of the ids
            bool done = false;
            for (int v = z.v0; v < z.v1 && !done; v += 32) {
                float l[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (v + lane < z.v1) z.line(v + lane, l);
                u64 w[4], part_sum = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int id = 4 * (v + lane) - lead + e;
                    w[e] = 0;
                    if (l[e] > -INFINITY && Sampler::inside(lim, order_key(l[e]), id)) {
                        const float f = z.weight(l[e]);
                        if (f >= min_p || l[e] == hi) w[e] = z.fixed(f);
                    }
                    part_sum += w[e];
                }
                u64 upto = part_sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                u64 c = before + upto - part_sum;
                if (c <= draw && draw < c + part_sum) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (c <= draw && draw < c + w[e]) {
                            token = 4 * (v + lane) - lead + e;
                            a.ids[row] = token;
                            if (a.logprobs) {
                                float t = 0.f;
                                for (uint32_t r = 0; r < ctas; ++r) t += *in_cta(&s.lp[r], r);
                                a.logprobs[row] = (l[e] == hi ? 0.f : l[e] - hi) - logf(t);
                            }
                        }
                        c += w[e];
                    }
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
                done = before > draw;
            }
        }
    } else {
        cluster_barrier();
        if (rank == 0 && tid == 0) {
            a.ids[row] = token;
            if (a.logprobs) {
                float t = 0.f;
                for (uint32_t r = 0; r < ctas; ++r) t += *in_cta(&s.lp[r], r);
                a.logprobs[row] = -logf(t);
            }
        }
    }
    cluster_barrier();    // nobody leaves while its shared memory may be read
}

}  // namespace dsuf

using namespace dsuf;

extern "C" int32_t dsuf_sample(dsuf_ctx* ctx, void* stream, uint64_t logits, int64_t ld, int32_t m, int32_t n, uint64_t temperature, uint64_t top_k,
                               uint64_t top_p, uint64_t min_p, uint64_t u, uint64_t ids_out, uint64_t logprobs_out) {
    if (!ctx) return DSUF_E_BADARG;
    DSUF_REQUIRE(ctx, m >= 0 && n >= 1 && n <= (1 << 22) && ld >= n, "sample: m >= 0, n in 1..2^22 (the weights' sum fits 64 bits), ld >= n");
    DSUF_REQUIRE(ctx, (long long)m * SA_MAX_CLUSTER <= 0x7fffffffll, "sample: too many rows");
    if (m == 0) return DSUF_OK;
    DSUF_REQUIRE(ctx, logits && u && ids_out && ((logits | u | ids_out | logprobs_out | temperature | top_k | top_p | min_p) & 3) == 0,
                 "sample: null or misaligned pointer");
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = (const float*)logits; a.ld = ld; a.n = n;
    a.temperature = (const float*)temperature; a.top_p = (const float*)top_p; a.min_p = (const float*)min_p; a.u = (const float*)u;
    a.top_k = (const int*)top_k; a.ids = (int*)ids_out; a.logprobs = (float*)logprobs_out;
    // as many CTAs per row as the GPU holds at once (two per SM), each with at least 2048 logits: fewer are not worth the cluster's barriers
    int c = SA_MAX_CLUSTER;
    while (c > 1 && ((long long)m * c > 2ll * ctx->sm_count || n < 2048 * c)) c >>= 1;
    return launch_cluster(ctx, (cudaStream_t)stream, sample_kernel, dim3(m * c), dim3(SA_THREADS), 0, c, a);
}
