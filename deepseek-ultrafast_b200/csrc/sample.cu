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
//   2. top-k: counts in 2048 bins of l (linear from M down, so that bins are evenly filled; a monotone map, so bins are an order).  The
//      tokens of the one bin where the limit falls are listed (usually some dozens) and ranked against each other: the limit becomes a
//      threshold (logit, id).  A bin with more than 512 tokens is split again by the bits of the logits, down to equal ones, of which
//      the id decides.
//   3. top-p: the same with weights, over the tokens inside the first limit (without top-k: all)
//   4. weight of C per warp, and the owner of the drawn number walks its part.
// What the CTAs tell each other is pushed into everybody's shared memory before a barrier, not fetched after it: a remote load costs
// about 250 cycles, and there are many.
// The exponent is formed in 64 bits ((l - M) / T rounded to fp32 would be off by 1e-6 relative in a far token's weight).
#include "internal.h"

namespace dsuf {

constexpr int SA_THREADS = 512;
constexpr int SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = 2048;
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
    uint32_t count[SA_BINS];                       // this CTA's histogram
    uint32_t mass_lo[SA_BINS], mass_hi[SA_BINS];
    uint32_t all_count[SA_BINS];                   // the row's
    u64 all_mass[SA_BINS];
    uint32_t list_key[SA_LIST];                    // this CTA's tokens of the limit's bin
    int list_id[SA_LIST];
    u64 row_at[SA_LIST];                           // the row's, as one word that orders them: key, then the complement of the id
    u64 row_w[SA_LIST];
    uint32_t n_list;
    uint32_t lists[SA_MAX_CLUSTER];
    float top[SA_MAX_CLUSTER], low[SA_MAX_CLUSTER], lp[SA_MAX_CLUSTER];
    int first[SA_MAX_CLUSTER];
    u64 kept[SA_MAX_CLUSTER];
    uint32_t key_hi[SA_MAX_CLUSTER], key_lo[SA_MAX_CLUSTER], ties[SA_MAX_CLUSTER];
    uint32_t own_hi, own_lo;
    u64 warp_a[SA_WARPS];
    uint32_t warp_b[SA_WARPS];
    float warp_f[SA_WARPS], warp_g[SA_WARPS];
    int found_bin;
    u64 found_mass, found_before;
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
    DSUF_DEV u64 block_sum(u64 v) {     // over the CTA, the result in every thread
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

    // The last token inside a limit: everything of a larger key is inside, and of this key the ids up to `id`.
    struct Limit {
        uint32_t key;
        int id;
        DSUF_DEV bool holds(uint32_t k, int i) const { return k > key || (k == key && i <= id); }
    };

    DSUF_DEV void clear_bins() {
        for (int i = tid; i < SA_BINS; i += SA_THREADS) s.count[i] = s.mass_lo[i] = s.mass_hi[i] = 0;
        __syncthreads();
    }
    DSUF_DEV void add(uint32_t b, u64 w, bool with_mass) {
        atomicAdd(&s.count[b], 1u);
        if (with_mass) {
            // a 64-bit sum in two words: the carry of the low one goes with the high one
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.mass_lo[b], lo);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
            if (hi) atomicAdd(&s.mass_hi[b], hi);
        }
    }
    // the CTAs' histograms, summed, into everybody's all_count / all_mass
    DSUF_DEV void share_bins(bool with_mass) {
        cluster_barrier();
        const int per = SA_BINS / ctas;
        for (int i = tid; i < per; i += SA_THREADS) {
            const int b = rank * per + i;
            uint32_t c[SA_MAX_CLUSTER], lo[SA_MAX_CLUSTER], hi[SA_MAX_CLUSTER];
#pragma unroll
            for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) {
                c[r] = lo[r] = hi[r] = 0;
                if (r < ctas) {
                    c[r] = ld_cluster_u32(&s.count[b], r);
                    if (with_mass) {
                        lo[r] = ld_cluster_u32(&s.mass_lo[b], r);
                        hi[r] = ld_cluster_u32(&s.mass_hi[b], r);
                    }
                }
            }
            uint32_t cs = 0;
            u64 ms = 0;
#pragma unroll
            for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) {
                cs += c[r];
                ms += ((u64)hi[r] << 32) + lo[r];
            }
            for (uint32_t r = 0; r < ctas; ++r) {
                *in_cta(&s.all_count[b], r) = cs;
                *in_cta(&s.all_mass[b], r) = ms;
            }
        }
        cluster_barrier();
    }
    // The bin where the limit falls (by count: the first where `want` tokens are reached, by weight: `target`), counting from count0 /
    // mass0, and what lies before it.
    DSUF_DEV void find_bin(bool by_mass, u64 want, double target, u64 count0, u64 mass0) {
        constexpr int PER = SA_BINS / SA_THREADS;
        u64 c[PER], cs = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int b = tid * PER + e;
            c[e] = by_mass ? s.all_mass[b] : s.all_count[b];
            cs += c[e];
        }
        u64 ci = cs;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 cv = __shfl_up_sync(0xffffffffu, ci, o);
            if (lane >= o) ci += cv;
        }
        __syncthreads();
        if (lane == 31) s.warp_a[warp] = ci;
        __syncthreads();
        u64 cb = (by_mass ? mass0 : count0) + ci - cs;
        for (int w = 0; w < warp; ++w) cb += s.warp_a[w];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const bool hit = by_mass ? (double)cb < target && target <= (double)(cb + c[e]) : cb < want && want <= cb + c[e];
            if (hit) {
                s.found_bin = tid * PER + e;
                s.found_before = cb;
                s.found_count = s.all_count[tid * PER + e];
            }
            cb += c[e];
        }
        __syncthreads();
    }

    // The limit inside the row's histogram of bin() over the tokens that `within` holds: `want` tokens, or the token whose weight, added to
    // that of all before it, reaches `target`.  One of the two exists: want is at most the number of tokens, target at most their weight.
    DSUF_DEV Limit limit(bool by_mass, u64 want, double target, const Limit within) {
        find_bin(by_mass, want, target, 0, 0);
        const int b0 = s.found_bin;
        u64 before = s.found_before;      // tokens, or weight, ahead of the bin
        uint32_t n_in = s.found_count, k_hi = 0xffffffffu, k_lo = 0;
        __syncthreads();
        auto mine = [&](int id, float l) {
            if (l == -INFINITY || bin(l) != b0) return false;
            const uint32_t k = order_key(l);
            return k >= k_lo && k <= k_hi && within.holds(k, id);
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
                if (tid == 0) { s.own_hi = 0; s.own_lo = 0xffffffffu; }
                __syncthreads();
                if (lane == 0) { atomicMax(&s.own_hi, hi); atomicMin(&s.own_lo, lo); }
                __syncthreads();
                if (tid < ctas) {
                    *in_cta(&s.key_hi[rank], tid) = s.own_hi;
                    *in_cta(&s.key_lo[rank], tid) = s.own_lo;
                }
                cluster_barrier();
                k_hi = 0; k_lo = 0xffffffffu;
                for (uint32_t r = 0; r < ctas; ++r) {
                    k_hi = max(k_hi, s.key_hi[r]);
                    k_lo = min(k_lo, s.key_lo[r]);
                }
                first_split = false;
            }
            int shift = 0;
            while (((k_hi - k_lo) >> shift) >= (uint32_t)SA_BINS) ++shift;
            cluster_barrier();               // (the others are through with this CTA's histogram)
            clear_bins();
            each([&](int id, float l) {
                if (mine(id, l)) add((k_hi - order_key(l)) >> shift, by_mass ? fixed(weight(l)) : 0, by_mass);
            });
            share_bins(by_mass);
            find_bin(by_mass, want, target, before, before);
            const uint32_t b = (uint32_t)s.found_bin;
            before = s.found_before;
            n_in = s.found_count;
            __syncthreads();
            k_hi -= b << shift;
            k_lo = max(k_lo, k_hi - min(k_hi, (1u << shift) - 1u));
        }
        Limit out;
        if (n_in <= SA_LIST) {
            // list the tokens, everybody gets them all, every thread ranks one or a share of one
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
            __syncthreads();
            if (tid < ctas) *in_cta(&s.lists[rank], tid) = min(s.n_list, (uint32_t)SA_LIST);
            cluster_barrier();
            uint32_t total = 0;
            for (uint32_t r = 0; r < ctas; ++r) {
                const uint32_t n = s.lists[r];
                // (the warps of a CTA take the lists in turn, so that their remote loads overlap)
                if (warp % ctas == r)
                    for (uint32_t i = (warp / ctas) * 32 + lane; i < n && total + i < SA_LIST; i += (SA_WARPS / ctas) * 32) {
                        const uint32_t k = ld_cluster_u32(&s.list_key[i], r);
                        s.row_at[total + i] = ((u64)k << 32) | (0xffffffffu - ld_cluster_u32(&s.list_id[i], r));
                        s.row_w[total + i] = by_mass ? fixed(weight(key_value(k))) : 1;
                    }
                total = min(total + n, (uint32_t)SA_LIST);
            }
            cluster_barrier();               // (nobody reads this CTA's list any more)
            int share = 1;                   // threads per token
            while (share < 32 && total * share * 2 <= SA_THREADS) share <<= 1;
            const uint32_t i = tid / share;
            const u64 mine_at = i < total ? s.row_at[i] : 0;
            u64 c = 0;
            for (uint32_t j = tid % share; j < total; j += share)
                if (s.row_at[j] > mine_at) c += s.row_w[j];
            for (int o = share >> 1; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            if (i < total && tid % share == 0) {
                c += before;
                const u64 after = c + s.row_w[i];
                if (by_mass ? (double)c < target && target <= (double)after : c < want && want <= after) {
                    s.found_key = (uint32_t)(mine_at >> 32);
                    s.found_id = (int)(0xffffffffu - (uint32_t)mine_at);
                }
            }
            __syncthreads();
            out.key = s.found_key;
            out.id = s.found_id;
            __syncthreads();
            return out;
        }
        // many equal logits: the r-th lowest id among them
        const u64 w = fixed(weight(key_value(k_hi)));
        u64 r = by_mass ? (u64)ceil((target - (double)before) / (double)(w ? w : 1)) : want - before;
        r = min(max(r, (u64)1), (u64)n_in);
        out.key = k_hi;
        uint32_t eq = 0;
        each([&](int id, float l) { eq += mine(id, l) ? 1u : 0u; });
        eq = __reduce_add_sync(0xffffffffu, eq);
        __syncthreads();
        if (lane == 0) s.warp_b[warp] = eq;
        __syncthreads();
        if (tid < ctas) {
            uint32_t t = 0;
            for (int q = 0; q < SA_WARPS; ++q) t += s.warp_b[q];
            *in_cta(&s.ties[rank], tid) = t;
        }
        cluster_barrier();
        u64 ahead = 0;
        for (uint32_t q = 0; q < rank; ++q) ahead += s.ties[q];
        for (int q = 0; q < warp; ++q) ahead += s.warp_b[q];
        if (ahead < r && r <= ahead + eq) {
            // this warp holds it: walk its lines in order
            for (int v = v0; v < v1; v += 32) {
                float l[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (v + lane < v1) line(v + lane, l);
                uint32_t n = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) n += mine(4 * (v + lane) - lead + e, l[e]) ? 1u : 0u;
                uint32_t upto = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                u64 at = ahead + upto - n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (mine(4 * (v + lane) - lead + e, l[e]) && ++at == r)
                        for (uint32_t q = 0; q < ctas; ++q) *in_cta(&s.found_id, q) = 4 * (v + lane) - lead + e;
                ahead += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        cluster_barrier();
        out.id = s.found_id;
        cluster_barrier();    // (a faster CTA's next limit does not write into found_id yet)
        return out;
    }
};

__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem);
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t rank = cluster_cta_rank(), ctas = cluster_num_ctas();
    const int row = blockIdx.x / ctas;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* x = a.logits + (size_t)row * a.ld;
    const int lead = (int)(((uintptr_t)x >> 2) & 3);
    const int lines = (int)(((long long)a.n + lead + 3) / 4);
    const long long parts = (long long)ctas * SA_WARPS, part = (long long)rank * SA_WARPS + warp;
    Sampler z{a, s, x, lead, (int)(lines * part / parts), (int)(lines * (part + 1) / parts), tid, warp, lane, rank, ctas, 0.f, 0.f, 0.0};
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
    if (tid < ctas) {
        for (int w = 0; w < SA_WARPS; ++w) {
            const float h = s.warp_f[w];
            const int i = (int)s.warp_b[w];
            if (w == 0 || h > hi || (h == hi && i < at)) { hi = h; at = i; }
            lo = w == 0 ? s.warp_g[w] : fminf(lo, s.warp_g[w]);
        }
        *in_cta(&s.top[rank], tid) = hi;
        *in_cta(&s.low[rank], tid) = lo;
        *in_cta(&s.first[rank], tid) = at;
    }
    cluster_barrier();
    hi = -INFINITY; lo = INFINITY; at = 0x7fffffff;
    for (uint32_t r = 0; r < ctas; ++r) {
        const float h = s.top[r];
        const int i = s.first[r];
        if (h > hi || (h == hi && i < at)) { hi = h; at = i; }
        lo = fminf(lo, s.low[r]);
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

    // ---- the limits; the first pass over all tokens also sums for the log-probability (temperature 1) ----
    bool want_lp = a.logprobs != nullptr;
    float lp = 0.f;
    u64 sum = 0;
    Sampler::Limit lim;
    lim.key = order_key(-INFINITY) + 1;    // every token above -inf
    lim.id = 0x7fffffff;
    if (!greedy && top_k > 0) {
        z.clear_bins();
        z.each([&](int id, float l) {
            if (l == -INFINITY) return;
            if (want_lp) lp += expf(l == hi ? 0.f : l - hi);
            z.add(z.bin(l), 0, false);
        });
        want_lp = false;
        z.share_bins(false);
        u64 tokens = 0;
        for (int i = tid; i < SA_BINS; i += SA_THREADS) tokens += s.all_count[i];
        if ((u64)top_k < z.block_sum(tokens)) lim = z.limit(false, (u64)top_k, 0.0, lim);
    }
    if (!greedy && top_p < 1.f) {
        if (top_k > 0) cluster_barrier();   // (the others are through with this CTA's histogram)
        z.clear_bins();
        z.each([&](int id, float l) {
            if (l == -INFINITY) return;
            if (want_lp) lp += expf(l == hi ? 0.f : l - hi);
            if (lim.holds(order_key(l), id)) z.add(z.bin(l), z.fixed(z.weight(l)), true);
        });
        want_lp = false;
        z.share_bins(true);
        u64 mass = 0;
        for (int i = tid; i < SA_BINS; i += SA_THREADS) mass += s.all_mass[i];
        // the first token is always inside: a target below one unit of weight is reached by it
        lim = z.limit(true, 0, fmax((double)top_p * (double)z.block_sum(mass), 0.5), lim);
    }
    if (!greedy || want_lp) {
        z.each([&](int id, float l) {
            if (l == -INFINITY) return;
            if (want_lp) lp += expf(l == hi ? 0.f : l - hi);
            if (!greedy && lim.holds(order_key(l), id)) {
                const float w = z.weight(l);
                if (w >= min_p || l == hi) sum += z.fixed(w);
            }
        });
    }
    if (a.logprobs) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lp += __shfl_xor_sync(0xffffffffu, lp, o);
        __syncthreads();
        if (lane == 0) s.warp_f[warp] = lp;
        __syncthreads();
        if (tid < ctas) {
            float t = 0.f;
            for (int w = 0; w < SA_WARPS; ++w) t += s.warp_f[w];
            *in_cta(&s.lp[rank], tid) = t;
        }
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
        if (tid < ctas) {
            u64 t = 0;
            for (int w = 0; w < SA_WARPS; ++w) t += s.warp_a[w];
            *in_cta(&s.kept[rank], tid) = t;
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
                    if (l[e] > -INFINITY && lim.holds(order_key(l[e]), id)) {
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
                                for (uint32_t r = 0; r < ctas; ++r) t += s.lp[r];
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
                for (uint32_t r = 0; r < ctas; ++r) t += s.lp[r];
                a.logprobs[row] = -logf(t);
            }
        }
    }
    cluster_barrier();    // nobody leaves while its shared memory may be read
}

int sample_setup(dsuf_ctx* ctx) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleShared));
    return e == cudaSuccess ? DSUF_OK : cuda_fail(ctx, e, "cudaFuncSetAttribute(sample)");
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
    return launch_cluster(ctx, (cudaStream_t)stream, sample_kernel, dim3(m * c), dim3(SA_THREADS), sizeof(SampleShared), c, a);
}
