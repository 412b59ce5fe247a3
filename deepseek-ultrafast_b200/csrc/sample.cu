// Token sampling from logits (dsuf_sample): temperature, top-k, top-p, min-p and one given uniform number per row.
//
// With M the largest logit of a row, weights w_i = exp((l_i - M) / T) and the order "larger logit first, lower id first among equals":
//   A = the first top_k tokens; B = those of A whose preceding weight inside A is below top_p * weight(A) (the first always);
//   C = those of B with w_i >= min_p (the first always); the drawn token is the lowest id i of C with weight(C, ids <= i) > u weight(C).
// The reference's sampler (crates/kernels/cu/sample.cu) merges the output head's records; this one works on the logits themselves, so that
// top_k and top_p have no limit.
//
// Nothing is sorted.  A cluster of up to 16 CTAs shares a row (latency-bound at few rows; the row comes from HBM once and from L2 in the
// later passes).  Weights are 40-bit fixed point, their sums 64-bit integers: exact, so the result depends neither on the split nor
// on the order of the histogram's atomics.  Passes:
//   1. the largest logit
//   2. top-k: counts in 2048 bins of l (linear from M down, so that bins are evenly filled; a monotone map, so bins are an order).  The
//      tokens of the one bin where the limit falls are listed (usually some dozens) and ranked against each other: the limit becomes a
//      threshold (logit, id).  A bin with more than 1024 tokens is split again by the bits of the logits, down to equal ones, of which
//      the id decides.
//   3. top-p: the same with weights, over the tokens inside the first limit (without top-k: all)
//   4. weight of C per warp, and the owner of the drawn number walks its part.
// Where all tokens down to the first limit's bin fit the list (the usual case: top_k up to about a thousand, or a peaked row), one CTA finishes
// from the list: ranks, both limits, min-p and the draw (129280 logits, top_k 50, top_p 0.9: 16 us instead of 38).
// What the CTAs tell each other is pushed into everybody's shared memory before a barrier, not fetched after it: a remote load costs
// about 250 cycles, and there are many.
// With many rows the passes are bound by instructions, not by bytes (64 rows of 129280 flat logits, top_p 0.9: 57 us, with the weights by scalar
// instructions 66, of which the largest logit took 5, weights and histogram 16, the list 8 and the kept weights 13; the histogram's atomics are 1 of it),
// so every pass computes no more than it needs.
// The exponent is carried in two fp32 numbers ((l - M) / T rounded to one would be off by 1e-6 relative in a far token's weight).
#include "internal.h"

namespace dsuf {

constexpr int SA_THREADS = 512;
constexpr int SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = 2048;
constexpr int SA_LIST = 1024;
constexpr int SA_MAX_CLUSTER = 16;
constexpr int SA_PER = SA_LIST / SA_THREADS;
constexpr int SA_FRACTION = 40;             // weight 1 in fixed point is 2^40
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
    uint32_t lo[SA_BINS], hi[SA_BINS];             // this CTA's histogram: counts (lo), or weights in two words
    u64 all[SA_BINS];                              // the row's
    uint32_t list_key[SA_LIST];                    // this CTA's tokens of the limit's bin
    int list_id[SA_LIST];
    u64 row_at[SA_LIST];                           // the row's, as one word that orders them: key, then the complement of the id
    u64 row_w[SA_LIST];
    uint32_t n_list;
    uint32_t lists[SA_MAX_CLUSTER];
    float top[SA_MAX_CLUSTER], lp[SA_MAX_CLUSTER];
    uint32_t tops[SA_MAX_CLUSTER], warp_tops[SA_WARPS];
    int first[SA_MAX_CLUSTER];
    u64 kept[SA_MAX_CLUSTER];
    uint32_t key_hi[SA_MAX_CLUSTER], key_lo[SA_MAX_CLUSTER], ties[SA_MAX_CLUSTER];
    uint32_t own_hi, own_lo;
    int own_first;
    u64 warp_a[SA_WARPS], warp_c[SA_WARPS];
    uint32_t warp_b[SA_WARPS];
    float warp_f[SA_WARPS];
    int found_bin;
    u64 found_before;
    uint32_t found_key;
    int found_id;
};

// The last token inside a limit: everything larger is inside, and of its equals the ids up to `id`.
struct Limit {
    float value;
    int id;
    DSUF_DEV bool holds(float l, int i) const { return l > value || (l == value && i <= id); }
};

struct Sampler {
    const SampleArgs& a;
    SampleShared& s;
    const float* x;          // the row
    int lead;                // elements between the 16-byte line of x[0] and x[0]
    int v0, v1;              // this warp's 16-byte lines
    int tid, warp, lane;
    uint32_t rank, ctas;
    float top, inv_bin, inv_temp, inv_temp_rest;   // inv_temp: log2(e) / T

    DSUF_DEV static float clean(float l) { return fmaxf(l, -INFINITY); }   // a NaN counts as -inf: never drawn
    DSUF_DEV void line(int v, float* l) const {
        const int i = 4 * v - lead;
#pragma unroll
        for (int e = 0; e < 4; ++e) l[e] = i + e >= 0 && i + e < a.n ? clean(x[i + e]) : -INFINITY;
    }
    // f(id, logit, the next id's logit) for all pairs of elements of this warp's part.  Lines that reach over the row's ends are read by elements (what
    // lies outside is -inf).  LIGHT: f is a few instructions, so four lines at a time; else one, with two more on their way (sixteen copies of a long f
    // do not stay in the instruction cache: 64 rows of 129280 logits, top_p 0.9, 70 us instead of 67; 16 rows 58 instead of 48).
    template <bool LIGHT = false, typename F>
    DSUF_DEV void each_pair(F f) const {
        const int full0 = lead > 0 ? 1 : 0, full1 = (a.n + lead) >> 2;
        const float4* lines = reinterpret_cast<const float4*>(x - lead);
        const int end = min(v1, full1);
        int v = max(v0, full0) + lane;
        auto four = [&](int w, float4 q) {
            f(4 * w - lead, clean(q.x), clean(q.y));
            f(4 * w - lead + 2, clean(q.z), clean(q.w));
        };
        if (LIGHT) {
            for (; v + 96 < end; v += 128) {
                float4 q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = lines[v + 32 * j];
#pragma unroll
                for (int j = 0; j < 4; ++j) four(v + 32 * j, q[j]);
            }
        }
        float4 q0 = v < end ? lines[v] : float4{}, q1 = v + 32 < end ? lines[v + 32] : float4{};
        for (; v < end; v += 32) {           // two lines ahead
            const float4 q = q0;
            q0 = q1;
            if (v + 64 < end) q1 = lines[v + 64];
            four(v, q);
        }
        if (lane < 2) {                      // lane 0: a cut first line, lane 1: a cut last one
            const int w = lane ? full1 : 0;
            const bool cut = lane ? ((a.n + lead) & 3) != 0 && !(full1 == 0 && full0) : full0 != 0;
            if (cut && w >= v0 && w < v1) {
                float l[4];
                line(w, l);
                for (int e = 0; e < 4; e += 2) f(4 * w - lead + e, l[e], l[e + 1]);
            }
        }
    }
    // f(id, logit)
    template <bool LIGHT = false, typename F>
    DSUF_DEV void each(F f) const {
        each_pair<LIGHT>([&](int id, float l0, float l1) {
            f(id, l0);
            f(id + 1, l1);
        });
    }
    // exp((l - top) / T) of two logits, by packed instructions.  The difference and the product are carried as unevaluated sums of two fp32 numbers
    // (Knuth's two-sum, an fma for the product's rest), because a rounding of the exponent is a relative error of the weight; the rests enter as a
    // factor 1 + rest.
    DSUF_DEV float2 weights(float l0, float l1) const {
        if (top == INFINITY) return make_float2(l0 == top ? 1.f : 0.f, l1 == top ? 1.f : 0.f);
        const u64 l = pack_f32x2(l0, l1), t = pack_f32x2(top, top), inv = pack_f32x2(inv_temp, inv_temp);
        const u64 d = sub2(l, t), v = sub2(d, l);
        const u64 rest = sub2(sub2(l, sub2(d, v)), add2(t, v));
        const u64 minus_z = mul2(d, pack_f32x2(-inv_temp, -inv_temp));
        const u64 z_rest = fma2(rest, inv, fma2(d, pack_f32x2(inv_temp_rest, inv_temp_rest), fma2(d, inv, minus_z)));
        const float2 y = unpack(mul2(z_rest, pack_f32x2(0.6931471805599453f, 0.6931471805599453f))), z = unpack(minus_z);
        float2 w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w.x) : "f"(-z.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w.y) : "f"(-z.y));
        return make_float2(z.x < 100.f ? fmaf(w.x, y.x, w.x) : 0.f, z.y < 100.f ? fmaf(w.y, y.y, w.y) : 0.f);
    }
    DSUF_DEV float weight(float l) const { return weights(l, l).x; }
    DSUF_DEV static float2 unpack(u64 v) {
        float2 r;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
        return r;
    }
    DSUF_DEV static u64 add2(u64 x, u64 y) { u64 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
    DSUF_DEV static u64 sub2(u64 x, u64 y) { u64 r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
    DSUF_DEV static u64 mul2(u64 x, u64 y) { u64 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
    DSUF_DEV static u64 fma2(u64 x, u64 y, u64 z) { u64 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z)); return r; }
    // w * 2^40, truncated
    DSUF_DEV static u64 fixed(float w) {
        return __float2ull_rz(w * (float)(1ull << SA_FRACTION));
    }
    // (rounding to the nearest bin by the addition's own rounding: any map that never goes up with the logit will do)
    DSUF_DEV int bin(float l) const {
        const float f = fminf(fmaxf((top - l) * inv_bin, 0.f), (float)(SA_BINS - 1));      // (inf - inf, inf * 0: NaN, so 0)
        return (int)(__float_as_uint(f + 8388608.f) & (SA_BINS - 1));
    }
    DSUF_DEV void clear_bins() {
        for (int i = tid; i < SA_BINS; i += SA_THREADS) s.lo[i] = s.hi[i] = 0;
        __syncthreads();
    }
    DSUF_DEV void add(uint32_t b, u64 w) {
        // a 64-bit sum in two words: the carry of the low one goes with the high one
        const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.lo[b], lo);
        const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&s.hi[b], hi);
    }
    // the CTAs' histograms, summed, into everybody's `all`
    DSUF_DEV void share_bins(bool two_words) {
        cluster_barrier();
        const int per = SA_BINS / ctas;
        for (int i = tid; i < per; i += SA_THREADS) {
            const int b = rank * per + i;
            uint32_t lo[SA_MAX_CLUSTER], hi[SA_MAX_CLUSTER];
#pragma unroll
            for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) {
                lo[r] = r < ctas ? ld_cluster_u32(&s.lo[b], r) : 0;
                hi[r] = r < ctas && two_words ? ld_cluster_u32(&s.hi[b], r) : 0;
            }
            u64 sum = 0;
#pragma unroll
            for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) sum += ((u64)hi[r] << 32) + lo[r];
            for (uint32_t r = 0; r < ctas; ++r) *in_cta(&s.all[b], r) = sum;
        }
        cluster_barrier();
    }
    // Whether an amount that goes from `from` to `to` is where the limit falls: the first to reach `want` tokens, or the weight `target`.
    DSUF_DEV static bool reaches(bool by_mass, u64 want, double target, u64 from, u64 to) {
        return by_mass ? (double)from < target && target <= (double)to : from < want && want <= to;
    }
    // Running sums over the row's bins: this thread's, the amount before them, and that of all.
    static constexpr int BINS_PER = SA_BINS / SA_THREADS;
    struct Scan {
        u64 c[BINS_PER], before, all;
    };
    DSUF_DEV Scan scan_bins() {
        Scan r;
        u64 cs = 0;
#pragma unroll
        for (int e = 0; e < BINS_PER; ++e) {
            r.c[e] = s.all[tid * BINS_PER + e];
            cs += r.c[e];
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
        r.before = ci - cs;
        r.all = 0;
#pragma unroll
        for (int w = 0; w < SA_WARPS; ++w) {
            const u64 v = s.warp_a[w];
            if (w < warp) r.before += v;
            r.all += v;
        }
        return r;
    }
    // The bin where the limit falls, counting from `start`, and the amount before it.
    DSUF_DEV int find_bin(const Scan& r, bool by_mass, u64 want, double target, u64& start) {
        u64 cb = start + r.before;
#pragma unroll
        for (int e = 0; e < BINS_PER; ++e) {
            if (reaches(by_mass, want, target, cb, cb + r.c[e])) {
                s.found_bin = tid * BINS_PER + e;
                s.found_before = cb;
            }
            cb += r.c[e];
        }
        __syncthreads();
        const int b = s.found_bin;
        start = s.found_before;
        __syncthreads();
        return b;
    }

    DSUF_DEV static uint32_t key(float l) { return order_key(l + 0.f); }     // (-0 orders as 0)
    // Lists this CTA's tokens that `take` wants (as far as there is room) and returns how many the row has.
    template <typename F>
    DSUF_DEV uint32_t list(F take) {
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        each([&](int id, float l) {
            if (take(id, l)) {
                const uint32_t at = atomicAdd(&s.n_list, 1u);
                if (at < SA_LIST) {
                    s.list_key[at] = key(l);
                    s.list_id[at] = id;
                }
            }
        });
        __syncthreads();
        if (tid < ctas) *in_cta(&s.lists[rank], tid) = s.n_list;
        cluster_barrier();
        uint32_t total = 0;
        for (uint32_t r = 0; r < ctas; ++r) total += s.lists[r];    // (at most n)
        return total;
    }
    // All CTAs' lists (at most SA_LIST tokens together) into row_at.  The warps take the CTAs in turn, so that their remote loads overlap.
    DSUF_DEV void fetch_list() {
        uint32_t base = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
            const uint32_t n = s.lists[r];
            if (warp % ctas == r)
                for (uint32_t i = (warp / ctas) * 32 + lane; i < n; i += (SA_WARPS / ctas) * 32)
                    s.row_at[base + i] = ((u64)ld_cluster_u32(&s.list_key[i], r) << 32) | (0xffffffffu - ld_cluster_u32(&s.list_id[i], r));
            base += n;
        }
    }
    // Sorts row_at (distinct words), largest first.  Up to 256 tokens by counting: a token's place is the number of larger ones, counted by
    // 2 to 32 threads of a warp (64 tokens: 0.5 us; a bitonic network, whose 21 steps each wait for shared memory twice, 3 us).  More by
    // a bitonic network (1024 tokens: 4 us against 20), where a warp's 32 pairs at distances up to 32 lie in 64 words of its own.
    DSUF_DEV void sort_list(uint32_t total) {
        __syncthreads();
        if (total <= 256) {
            uint32_t bits = 1;
            while (bits < 5 && (total << (bits + 1)) <= SA_THREADS) ++bits;
            const uint32_t share = 1u << bits, first = tid & (share - 1), i = tid >> bits;
            const u64 at = i < total ? s.row_at[i] : ~0ull;
            uint32_t place = 0;
            if ((uint32_t)(tid & ~31) >> bits < total) {
#pragma unroll 4
                for (uint32_t j = first; j < total; j += share) place += s.row_at[j] > at ? 1u : 0u;
                for (uint32_t o = share >> 1; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
            }
            __syncthreads();
            if (first == 0 && i < total) s.row_at[place] = at;
            __syncthreads();
            return;
        }
        uint32_t n = 512;
        while (n < total) n <<= 1;
        for (uint32_t i = total + tid; i < n; i += SA_THREADS) s.row_at[i] = 0;     // (below every token)
        __syncthreads();
        for (uint32_t k = 2; k <= n; k <<= 1)
            for (uint32_t j = k >> 1; j > 0; j >>= 1) {
                if (tid < n / 2) {
                    const uint32_t lo = tid + (tid & ~(j - 1)), hi = lo + j;      // the pairs of distance j, numbered by tid
                    const u64 p = s.row_at[lo], q = s.row_at[hi];
                    if ((p < q) == ((lo & k) == 0)) {
                        s.row_at[lo] = q;
                        s.row_at[hi] = p;
                    }
                }
                if (j > 32 || (j == 1 && k >= 64)) __syncthreads();
                else __syncwarp();
            }
    }
    // Sums of what the earlier threads, and this thread earlier, hold (w: SA_PER values of each).
    DSUF_DEV u64 block_ahead(const u64* w, u64* ahead) {
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < SA_PER; ++e) own += w[e];
        u64 upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        __syncthreads();
        if (lane == 31) s.warp_a[warp] = upto;
        __syncthreads();
        u64 at = upto - own, all = 0;
#pragma unroll
        for (int q = 0; q < SA_WARPS; ++q) {
            if (q < warp) at += s.warp_a[q];
            all += s.warp_a[q];
        }
#pragma unroll
        for (int e = 0; e < SA_PER; ++e) {
            ahead[e] = at;
            at += w[e];
        }
        return all;
    }
    // The whole rest of a row whose candidates are all listed (one CTA): the first `want` of the order, of these the ones whose preceding weight
    // is below top_p of `mass` (0: of their own), of these min_p, and the draw.
    template <typename F>
    DSUF_DEV void finish(uint32_t total, u64 want, float top_p, u64 mass, float min_p, float u, F store) {
        sort_list(total);
        float l[SA_PER], f[SA_PER];
        u64 w[SA_PER], ahead[SA_PER];
        uint32_t id[SA_PER];
#pragma unroll
        for (int e = 0; e < SA_PER; ++e) {
            const uint32_t i = tid * SA_PER + e;
            const bool in = i < total && i < want;
            const u64 at = in ? s.row_at[i] : 0;
            id[e] = 0xffffffffu - (uint32_t)at;
            l[e] = key_value((uint32_t)(at >> 32));
            f[e] = in ? weight(l[e]) : 0.f;
            w[e] = in ? fixed(f[e]) : 0;
        }
        const u64 own = block_ahead(w, ahead);
        const double target = top_p < 1.f ? fmax((double)top_p * (double)(mass ? mass : own), 0.5) : INFINITY;
        // the tokens that stay, in the order of their ids
        if (tid == 0) s.n_list = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < SA_PER; ++e) {
            s.row_w[tid * SA_PER + e] = w[e];
            if (w[e] && (double)ahead[e] < target && f[e] >= min_p)
                s.row_at[atomicAdd(&s.n_list, 1u)] = ((u64)(0xffffffffu - id[e]) << 32) | (uint32_t)(tid * SA_PER + e);
        }
        __syncthreads();
        const uint32_t stay = s.n_list;
        sort_list(stay);
#pragma unroll
        for (int e = 0; e < SA_PER; ++e) {
            const uint32_t i = tid * SA_PER + e;
            w[e] = i < stay ? s.row_w[(uint32_t)s.row_at[i]] : 0;
        }
        const u64 kept = block_ahead(w, ahead);
        u64 draw = u > 0.f ? (u64)((double)u * (double)kept) : 0;
        draw = min(draw, kept - 1);
#pragma unroll
        for (int e = 0; e < SA_PER; ++e)
            if (ahead[e] <= draw && draw < ahead[e] + w[e]) {
                const uint32_t token = 0xffffffffu - (uint32_t)(s.row_at[tid * SA_PER + e] >> 32);
                store((int)token, clean(x[token]));
            }
    }

    // The limit inside the row's histogram of bin() over the tokens that `within` holds: `want` tokens, or the token whose weight, added to
    // that of all before it, reaches `target`.  One of the two exists: want is at most the number of tokens, target at most their weight.
    // b0: the bin where it falls, before: tokens, or weight, ahead of it.
    DSUF_DEV Limit limit(bool by_mass, u64 want, double target, const Limit within, int b0, u64 before) {
        uint32_t k_hi = 0xffffffffu, k_lo = 0;
        auto mine = [&](int id, float l) {
            if (bin(l) != b0 || !within.holds(l, id)) return false;
            const uint32_t k = key(l);
            return k >= k_lo && k <= k_hi;
        };
        for (bool first_split = true;; first_split = false) {
            // everybody gets the bin's tokens, every thread ranks some or a share of one
            const uint32_t total = list(mine);
            if (total <= SA_LIST) {
                fetch_list();
                cluster_barrier();               // (nobody reads this CTA's list any more)
                sort_list(total);
                u64 w[SA_PER], ahead[SA_PER];
#pragma unroll
                for (int e = 0; e < SA_PER; ++e) {
                    const uint32_t i = tid * SA_PER + e;
                    w[e] = i < total ? by_mass ? fixed(weight(key_value((uint32_t)(s.row_at[i] >> 32)))) : 1 : 0;
                }
                block_ahead(w, ahead);
#pragma unroll
                for (int e = 0; e < SA_PER; ++e) {
                    const uint32_t i = tid * SA_PER + e;
                    if (i < total && reaches(by_mass, want, target, before + ahead[e], before + ahead[e] + w[e])) {
                        s.found_key = (uint32_t)(s.row_at[i] >> 32);
                        s.found_id = (int)(0xffffffffu - (uint32_t)s.row_at[i]);
                    }
                }
                __syncthreads();
                const Limit out = {key_value(s.found_key), s.found_id};
                __syncthreads();
                return out;
            }
            if (k_hi == k_lo) break;
            // too many: split the bin by its logits' bits
            if (first_split) {
                uint32_t hi = 0, lo = 0xffffffffu;
                each([&](int id, float l) {
                    if (mine(id, l)) {
                        hi = max(hi, key(l));
                        lo = min(lo, key(l));
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
            }
            int shift = 0;
            while (((k_hi - k_lo) >> shift) >= (uint32_t)SA_BINS) ++shift;
            clear_bins();      // (the others read this CTA's histogram before the last barrier)
            each([&](int id, float l) {
                if (mine(id, l)) add((k_hi - key(l)) >> shift, by_mass ? fixed(weight(l)) : 1);
            });
            share_bins(by_mass);
            const uint32_t b = (uint32_t)find_bin(scan_bins(), by_mass, want, target, before);
            k_hi -= b << shift;
            k_lo = max(k_lo, k_hi - min(k_hi, (1u << shift) - 1u));
        }
        // many equal logits: the r-th lowest id among them
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
        u64 ahead = 0, all = 0;
        for (uint32_t q = 0; q < ctas; ++q) {
            if (q < rank) ahead += s.ties[q];
            all += s.ties[q];
        }
        for (int q = 0; q < warp; ++q) ahead += s.warp_b[q];
        const u64 w = fixed(weight(key_value(k_hi)));
        u64 r = by_mass ? (u64)ceil((target - (double)before) / (double)(w ? w : 1)) : want - before;
        r = min(max(r, (u64)1), all);
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
        const Limit out = {key_value(k_hi), s.found_id};
        cluster_barrier();    // (a faster CTA's next limit does not write into found_id yet)
        return out;
    }
};

__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem);
    cluster_arrive();        // (waited for before the first write into a peer's shared memory: the peer has to have started)
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t rank = cluster_cta_rank(), ctas = cluster_num_ctas();
    const int row = blockIdx.x / ctas;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* x = a.logits + (size_t)row * a.ld;
    const int lead = (int)(((uintptr_t)x >> 2) & 3);
    const int lines = (a.n + lead + 3) / 4;
    const long long parts = (long long)ctas * SA_WARPS, part = (long long)rank * SA_WARPS + warp;
    Sampler z{a, s, x, lead, (int)(lines * part / parts), (int)(lines * (part + 1) / parts), tid, warp, lane, rank, ctas, 0.f, 0.f, 0.f, 0.f};
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;      // (the top's weight is 1: it always stays)
    const bool greedy = !(temp > 0.f);

    // ---- the largest logit ----
    float hi = -INFINITY;
    z.each<true>([&](int id, float l) { hi = fmaxf(hi, l); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    if (lane == 0) s.warp_f[warp] = hi;
    if (tid == 0) s.own_first = 0x7fffffff;
    __syncthreads();
    cluster_wait();
    if (tid < ctas) {
        for (int w = 0; w < SA_WARPS; ++w) hi = fmaxf(hi, s.warp_f[w]);
        *in_cta(&s.top[rank], tid) = hi;
    }
    cluster_barrier();
    hi = -INFINITY;
    for (uint32_t r = 0; r < ctas; ++r) hi = fmaxf(hi, s.top[r]);
    z.top = hi;
    if (hi == -INFINITY) {    // nothing to draw from
        if (rank == 0 && tid == 0) {
            a.ids[row] = -1;
            if (a.logprobs) a.logprobs[row] = -INFINITY;
        }
        return;               // (all CTAs of the row alike, and nobody reads remote memory any more)
    }
    const double inv = greedy ? 1.0 : 1.4426950408889634 / (double)temp;
    z.inv_temp = (float)fmin(inv, 3.4028234663852886e38);      // (finite, so that the top's weight is 1 at any temperature)
    z.inv_temp_rest = inv > 3.4028234663852886e38 ? 0.f : (float)(inv - (double)z.inv_temp);
    const float span = fmaxf(24.f, 32.f * temp);
    z.inv_bin = span < INFINITY ? (float)(SA_BINS - 1) / span : 0.f;

    // ---- the limits; the first pass over all tokens also sums for the log-probability (temperature 1) ----
    bool want_lp = a.logprobs != nullptr;
    // (the largest logits are counted and the others summed: the logarithm of a sum next to 1 would lose what the others add to it)
    float lp = 0.f;
    uint32_t tops = 0;
    auto add_lp = [&](float l) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((l - hi) * 1.4426950408889634f));
        if (l == hi) ++tops;
        else lp += e;
    };
    // this CTA's sum into everybody's table; visible behind the next cluster barrier
    auto share_lp = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lp += __shfl_xor_sync(0xffffffffu, lp, o);
        tops = __reduce_add_sync(0xffffffffu, tops);
        __syncthreads();
        if (lane == 0) {
            s.warp_f[warp] = lp;
            s.warp_tops[warp] = tops;
        }
        __syncthreads();
        if (tid < ctas) {
            float t = 0.f;
            uint32_t n = 0;
            for (int w = 0; w < SA_WARPS; ++w) {
                t += s.warp_f[w];
                n += s.warp_tops[w];
            }
            *in_cta(&s.lp[rank], tid) = t;
            *in_cta(&s.tops[rank], tid) = n;
        }
    };
    auto store = [&](int token, float l) {
        a.ids[row] = token;
        if (a.logprobs) {
            float t = 0.f;
            uint32_t n = 0;
            for (uint32_t r = 0; r < ctas; ++r) {
                t += s.lp[r];
                n += s.tops[r];
            }
            a.logprobs[row] = fminf(l - hi, 0.f) - log1pf((float)(n - 1) + t);
        }
    };
    if (greedy) {
        int at = 0x7fffffff;
        if (want_lp)
            z.each([&](int id, float l) { add_lp(l); if (l == hi) at = min(at, id); });
        else
            z.each<true>([&](int id, float l) { if (l == hi) at = min(at, id); });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) atomicMin(&s.own_first, at);
        if (want_lp) share_lp();
        __syncthreads();
        if (tid < ctas) *in_cta(&s.first[rank], tid) = s.own_first;
        cluster_barrier();
        if (rank == 0 && tid == 0) {
            at = 0x7fffffff;
            for (uint32_t r = 0; r < ctas; ++r) at = min(at, s.first[r]);
            store(at, hi);
        }
        return;
    }
    const float u = a.u[row];
    u64 sum = 0;
    Limit lim = {-INFINITY, -1};           // every token above -inf
    bool cut = false;
    if (top_k > 0) {
        z.clear_bins();
        if (want_lp)
            z.each([&](int id, float l) { add_lp(l); if (l > -INFINITY) atomicAdd(&s.lo[z.bin(l)], 1u); });
        else
            z.each([&](int id, float l) { if (l > -INFINITY) atomicAdd(&s.lo[z.bin(l)], 1u); });
        if (want_lp) share_lp();
        want_lp = false;
        z.share_bins(false);
        const Sampler::Scan bins = z.scan_bins();
        cut = (u64)top_k < bins.all;
        if (cut) {
            u64 before = 0;
            const int b = z.find_bin(bins, false, (u64)top_k, 0.0, before);
            if (before + s.all[b] <= SA_LIST) {
                const uint32_t total = z.list([&](int id, float l) { return l > -INFINITY && z.bin(l) <= b; });
                if (rank == 0) z.fetch_list();
                cluster_arrive();        // (the other CTAs stay until their lists have been read)
                if (rank == 0) z.finish(total, (u64)top_k, top_p, 0, min_p, u, store);
                cluster_wait();
                return;
            }
            lim = z.limit(false, (u64)top_k, 0.0, lim, b, before);
        }
    }
    const bool few = cut;                  // the limits leave so little of the row that most warps meet none of it: they skip the weights
    if (top_p < 1.f) {
        z.clear_bins();    // (the others read this CTA's histogram before the last barrier)
        if (few)
            z.each([&](int id, float l) { if (lim.holds(l, id)) z.add(z.bin(l), z.fixed(z.weight(l))); });
        else
            z.each_pair([&](int id, float l0, float l1) {
                if (want_lp) {
                    add_lp(l0);
                    add_lp(l1);
                }
                const float2 w = z.weights(l0, l1);
                z.add(z.bin(l0), z.fixed(w.x));
                z.add(z.bin(l1), z.fixed(w.y));
            });
        if (want_lp) share_lp();
        want_lp = false;
        z.share_bins(true);
        // the first token is always inside: a target below one unit of weight is reached by it
        const Sampler::Scan bins = z.scan_bins();
        const u64 mass = bins.all;
        const double target = fmax((double)top_p * (double)mass, 0.5);
        u64 before = 0;
        const int b = z.find_bin(bins, true, 0, target, before);
        // Every token down to bin b weighs at least what the bin's edge does, which bounds their number; of flat rows the bound is near the
        // truth and far above the list's size: they do not try.
        const float edge = z.weight(hi - (float)(b + 1) / z.inv_bin);
        if (!cut && (double)(before + s.all[b]) <= 4.0 * SA_LIST * (double)z.fixed(edge)) {
            const uint32_t total = z.list([&](int id, float l) { return l > -INFINITY && z.bin(l) <= b; });
            if (total <= SA_LIST) {
                if (rank == 0) z.fetch_list();
                cluster_arrive();
                if (rank == 0) z.finish(total, ~0ull, top_p, mass, min_p, u, store);
                cluster_wait();
                return;
            }
            cluster_barrier();    // (everybody has read the lists' lengths: the next ones may be written)
        }
        lim = z.limit(true, 0, target, lim, b, before);
        cut = true;
    }
    if (few) {
        z.each([&](int id, float l) {
            if (lim.holds(l, id)) {
                const float w = z.weight(l);
                if (w >= min_p) sum += z.fixed(w);
            }
        });
    } else if (cut) {
        z.each_pair([&](int id, float l0, float l1) {
            const float2 w = z.weights(l0, l1);
            if (lim.holds(l0, id) && w.x >= min_p) sum += z.fixed(w.x);
            if (lim.holds(l1, id + 1) && w.y >= min_p) sum += z.fixed(w.y);
        });
    } else {
        z.each_pair([&](int id, float l0, float l1) {
            if (want_lp) {
                add_lp(l0);
                add_lp(l1);
            }
            const float2 w = z.weights(l0, l1);
            sum += (w.x >= min_p ? z.fixed(w.x) : 0) + (w.y >= min_p ? z.fixed(w.y) : 0);
        });
        if (want_lp) share_lp();
    }

    // ---- the draw ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) s.warp_a[warp] = sum;
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
    u64 draw = u > 0.f ? (u64)((double)u * (double)total) : 0;
    draw = min(draw, total - 1);
    if (draw < before || draw >= before + s.kept[rank]) return;
    // This CTA holds the token.  The part of the warp that holds it is dealt to all warps, then the warp of that share walks it in the order
    // of the ids.
    auto mass = [&](int id, float l) {
        if (!lim.holds(l, id)) return (u64)0;
        const float w = z.weight(l);
        return w >= min_p ? z.fixed(w) : 0;
    };
    int holder = 0;
    while (before + s.warp_a[holder] <= draw) before += s.warp_a[holder++];
    const long long p0 = lines * ((long long)rank * SA_WARPS + holder) / parts, p1 = lines * ((long long)rank * SA_WARPS + holder + 1) / parts;
    const int w0 = (int)(p0 + (p1 - p0) * warp / SA_WARPS), w1 = (int)(p0 + (p1 - p0) * (warp + 1) / SA_WARPS);
    u64 share = 0;
    for (int v = w0 + lane; v < w1; v += 32) {
        float l[4];
        z.line(v, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) share += mass(4 * v - lead + e, l[e]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) share += __shfl_xor_sync(0xffffffffu, share, o);
    if (lane == 0) s.warp_c[warp] = share;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += s.warp_c[w];
    if (draw < before || draw >= before + share) return;
    for (int v = w0; v < w1 && before <= draw; v += 32) {
        float l[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (v + lane < w1) z.line(v + lane, l);
        u64 w[4], here = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = mass(4 * (v + lane) - lead + e, l[e]);
            here += w[e];
        }
        u64 upto = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        u64 c = before + upto - here;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (c <= draw && draw < c + w[e]) store(4 * (v + lane) - lead + e, l[e]);
            c += w[e];
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
}

int sample_setup(dsuf_ctx* ctx) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleShared));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);   // clusters of 16
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
    const uint64_t bytes = 4ull * m;
    auto meets = [&](uint64_t x, uint64_t y) { return x && y && x < y + bytes && y < x + bytes; };
    bool apart = !meets(ids_out, logprobs_out);
    for (uint64_t o : {ids_out, logprobs_out}) {
        // (a row reads its settings before its result is written, so one of their columns may receive it)
        for (uint64_t c : {temperature, top_k, top_p, min_p, u}) apart = apart && (o == c || !meets(o, c));
        apart = apart && !(o && block_meets_rows(o, (long long)bytes, logits, 2 * ld, 2ll * n, m));      // (rows of n fp32: 2 n halves)
    }
    DSUF_REQUIRE(ctx, apart, "sample: ids and logprobs must share no memory with the logits, each other or (but for a whole column) the settings");
    DSUF_REQUIRE_DEVICE(ctx, "sample");
    SampleArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = (const float*)logits; a.ld = ld; a.n = n;
    a.temperature = (const float*)temperature; a.top_p = (const float*)top_p; a.min_p = (const float*)min_p; a.u = (const float*)u;
    a.top_k = (const int*)top_k; a.ids = (int*)ids_out; a.logprobs = (float*)logprobs_out;
    // As many CTAs per row as the GPU holds at once (two per SM), each with at least 2048 logits: fewer are not worth the cluster's barriers.
    // Clusters of 16 only while four fifths of the SMs hold them all: a cluster lies inside one GPC, which has room for one of 16 and some rest, so
    // with more of them CTAs share SMs (129280 logits, top_k 50, top_p 0.9; 16 against 8: 1 row 15.3 / 17.1 us, 7 rows 15.6 / 17.3, 8 rows
    // 19.4 / 17.5, 16 rows 29.2 / 22.6; rows of mixed settings lose up to 5 % at 8 to 11 rows of that width and win as much or more elsewhere).
    int c = SA_MAX_CLUSTER;
    auto fits = [&](int cl) { return 5ll * m * cl <= (cl == SA_MAX_CLUSTER ? 4ll : 10ll) * ctx->sm_count; };
    while (c > 1 && (!fits(c) || n < 2048 * c)) c >>= 1;
    return launch_cluster(ctx, (cudaStream_t)stream, sample_kernel, dim3(m * c), dim3(SA_THREADS), sizeof(SampleShared), c, a);
}
