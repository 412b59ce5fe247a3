// Paged key/value cache: the write of new tokens, with the rotary embedding applied on the way (dsuf_kv_append).
//
// One pass: every 16-byte vector (8 columns of one head of one token) is read once, rotated in fp32 if it lies in the rotated
// columns, and written once -- q to q_out, k and v to their slot, as bf16 or as e4m3(x / scale).  HBM-bound: 2 bytes in and 2
// (or 1) out per element; the tables add 8 bytes per pair and token.  A CTA serves one token (or a share of its heads when
// tokens are few), and a thread keeps the same 8 columns for all its heads, so the cosines, sines, page lookup and position
// are fetched once per thread; the first three heads' loads are issued ahead of that chain of lookups.
// 16384 tokens, 56 + 2 x 8 heads of 128 into an e4m3 cache: 97 us = 5.9 TB/s, 0.91 of the measured copy bandwidth (CTAs of 64 threads with
// five heads per thread: 98 us, and 0.2 us more for the 64 tokens of a decode step, which take 2.3).
#include "internal.h"

namespace dsuf {

constexpr int KID_APPEND = 7;
constexpr int AP_THREADS = 128;
constexpr int AP_BATCH = 3;   // heads of a thread whose loads are issued together

struct AppendArgs {
    const bf16 *q, *k, *v;
    bf16 *q_out, *k_out;
    int ldq, ldk, ldv, ldqo, ldko;
    int q_heads, kv_heads, n_seqs, max_pages, n_pages, page_shift;
    const int *pos, *seq, *table;
    uint8_t *ck, *cv;
    const float *k_scale, *v_scale;
    long long page_stride;
    const float *cos, *sin;
    int rope_rows, rot, off;
    DevStatus* status;
};

// The 8 columns of `x` turned by the angles of cs / sn; `other`: the 8 columns they are paired with in the half form.
DSUF_DEV void rotate8(float* x, const float* other, const float* cs, const float* sn, bool half, bool second) {
    if (!half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * cs[i] - b * sn[i];
            x[2 * i + 1] = b * cs[i] + a * sn[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = second ? x[i] * cs[i] + other[i] * sn[i] : x[i] * cs[i] - other[i] * sn[i];
    }
}

DSUF_DEV void unpack8(uint4 u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
DSUF_DEV uint4 pack8(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// HALF: pairs rot / 2 apart (a kernel of its own, as the exchange costs the other form 10 registers and with them resident CTAs: 104 us instead of 97).
template <int D, bool FP8, bool HALF>
__global__ void __launch_bounds__(AP_THREADS) kv_append_kernel(const AppendArgs a) {
    constexpr int LANES = D / 8;                 // threads of one head
    constexpr int HPC = AP_THREADS / LANES;      // heads a CTA handles at a time
    pdl_wait();
    pdl_launch_dependents();
    const int tok = blockIdx.x;
    const int c8 = threadIdx.x % LANES;          // columns 8 c8 ..
    const int H = a.q_heads + 2 * a.kv_heads;
    // heads in the order q, k, v; the CTAs of one token deal them out
    uint4 raw[AP_BATCH];
    auto load = [&](int h0) {
#pragma unroll
        for (int j = 0; j < AP_BATCH; ++j) {
            const int h = h0 + j * gridDim.y * HPC + threadIdx.x / LANES;
            const bf16* src = nullptr;
            if (h < a.q_heads) src = a.q + (size_t)tok * a.ldq + (size_t)h * D;
            else if (h < a.q_heads + a.kv_heads) src = a.k + (size_t)tok * a.ldk + (size_t)(h - a.q_heads) * D;
            else if (h < H) src = a.v + (size_t)tok * a.ldv + (size_t)(h - a.q_heads - a.kv_heads) * D;
            raw[j] = src ? *reinterpret_cast<const uint4*>(src + c8 * 8) : make_uint4(0, 0, 0, 0);
        }
    };
    load(blockIdx.y * HPC);      // ahead of the chain position -> page -> slot, which only the stores need
    const int pos = a.pos[tok], seq = a.seq ? a.seq[tok] : tok;
    if (pos < 0 || seq < 0) return;   // padding
    const int page_i = pos >> a.page_shift;
    if (seq >= a.n_seqs || page_i >= a.max_pages || (a.rot && pos >= a.rope_rows)) {
        if (threadIdx.x == 0) report(a.status, DEVERR_BAD_PLAN, KID_APPEND, 1);
        return;
    }
    const int page = a.table[(size_t)seq * a.max_pages + page_i];
    if (page < 0 || page >= a.n_pages) {
        if (threadIdx.x == 0) report(a.status, DEVERR_BAD_PLAN, KID_APPEND, 2);
        return;
    }
    const int rel = c8 * 8 - a.off;
    const bool turn = rel >= 0 && rel < a.rot;
    const bool second = turn && rel >= a.rot / 2;   // half form: the second member of the pairs
    float cs[8], sn[8];
    if (turn) {
        const int i0 = HALF ? rel - (second ? a.rot / 2 : 0) : rel / 2;
        const int n4 = HALF ? 2 : 1;
        const float4* cp = reinterpret_cast<const float4*>(a.cos + (size_t)pos * (a.rot / 2) + i0);
        const float4* sp = reinterpret_cast<const float4*>(a.sin + (size_t)pos * (a.rot / 2) + i0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (j < n4) {
                const float4 c = __ldg(cp + j), s = __ldg(sp + j);
                cs[4 * j] = c.x; cs[4 * j + 1] = c.y; cs[4 * j + 2] = c.z; cs[4 * j + 3] = c.w;
                sn[4 * j] = s.x; sn[4 * j + 1] = s.y; sn[4 * j + 2] = s.z; sn[4 * j + 3] = s.w;
            }
        }
    }
    const int partner = HALF ? (second ? -a.rot / 16 : a.rot / 16) : 0;   // lanes to the other member of the pair
    const size_t slot = (size_t)(pos & ((1 << a.page_shift) - 1));
    for (int h0 = blockIdx.y * HPC; h0 < H; h0 += gridDim.y * HPC * AP_BATCH) {
        if (h0 >= (int)(gridDim.y * HPC * AP_BATCH)) load(h0);
#pragma unroll
        for (int j = 0; j < AP_BATCH; ++j) {
            const int h = h0 + j * gridDim.y * HPC + threadIdx.x / LANES;
            float x[8];
            unpack8(raw[j], x);
            if constexpr (HALF) {
                // every lane of the warp takes part; lanes outside the rotated columns read themselves
                const int from = (threadIdx.x & 31) + (turn ? partner : 0);
                uint4 o;
                o.x = __shfl_sync(0xffffffffu, raw[j].x, from);
                o.y = __shfl_sync(0xffffffffu, raw[j].y, from);
                o.z = __shfl_sync(0xffffffffu, raw[j].z, from);
                o.w = __shfl_sync(0xffffffffu, raw[j].w, from);
                if (turn && h < a.q_heads + a.kv_heads) {
                    float other[8];
                    unpack8(o, other);
                    rotate8(x, other, cs, sn, true, second);
                }
            } else if (turn && h < a.q_heads + a.kv_heads) {
                rotate8(x, nullptr, cs, sn, false, false);
            }
            if (h < a.q_heads) {
                *reinterpret_cast<uint4*>(a.q_out + (size_t)tok * a.ldqo + (size_t)h * D + c8 * 8) = pack8(x);
            } else if (h < H) {
                const bool is_v = h >= a.q_heads + a.kv_heads;
                const int kh = h - a.q_heads - (is_v ? a.kv_heads : 0);
                const size_t at = (size_t)page * a.page_stride + ((((size_t)kh << a.page_shift) + slot) * D + c8 * 8);
                uint8_t* dst = is_v ? a.cv : a.ck;
                if (!is_v && a.k_out) *reinterpret_cast<uint4*>(a.k_out + (size_t)tok * a.ldko + (size_t)kh * D + c8 * 8) = pack8(x);
                if constexpr (FP8) {
                    const float* sc = is_v ? a.v_scale : a.k_scale;
                    const float s = sc ? __ldg(sc + kh) : 1.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = x[i] / s;
                    *reinterpret_cast<uint2*>(dst + at) = make_uint2(f32x4_to_e4m3x4(x[0], x[1], x[2], x[3]), f32x4_to_e4m3x4(x[4], x[5], x[6], x[7]));
                } else {
                    *reinterpret_cast<uint4*>(dst + at * 2) = pack8(x);
                }
            }
        }
    }
}

int check_kv_cache(dsuf_ctx* ctx, const char* who, const dsuf_kv_cache* c) {
    DSUF_REQUIRE(ctx, c, "%s: null cache", who);
    DSUF_REQUIRE(ctx, c->dtype == DSUF_KV_BF16 || c->dtype == DSUF_KV_E4M3, "%s: unknown cache dtype %d", who, c->dtype);
    DSUF_REQUIRE(ctx, c->head_dim == 64 || c->head_dim == 128, "%s: head_dim (%d) must be 64 or 128", who, c->head_dim);
    DSUF_REQUIRE(ctx, c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
                 "%s: page_size (%d) must be a power of two in 16..1024", who, c->page_size);
    DSUF_REQUIRE(ctx, c->kv_heads >= 1 && c->kv_heads <= 1024 && c->n_pages >= 1, "%s: kv_heads (%d) must be in 1..1024 and n_pages (%d) positive", who,
                 c->kv_heads, c->n_pages);
    DSUF_REQUIRE(ctx, c->page_stride >= (int64_t)c->kv_heads * c->page_size * c->head_dim && c->page_stride % 16 == 0,
                 "%s: page_stride (%lld) must be a multiple of 16 and hold kv_heads * page_size * head_dim elements", who, (long long)c->page_stride);
    DSUF_REQUIRE(ctx, c->k && c->v && (c->k & 15) == 0 && (c->v & 15) == 0, "%s: k and v must be 16-byte aligned", who);
    DSUF_REQUIRE(ctx, c->dtype == DSUF_KV_E4M3 || (!c->k_scale && !c->v_scale), "%s: scales belong to an E4M3 cache", who);
    DSUF_REQUIRE(ctx, (c->k_scale & 3) == 0 && (c->v_scale & 3) == 0, "%s: misaligned scales", who);
    return DSUF_OK;
}

}  // namespace dsuf

using namespace dsuf;

extern "C" int32_t dsuf_kv_append(dsuf_ctx* ctx, void* stream, const dsuf_kv_cache* cache, uint64_t k, int32_t ldk, uint64_t v, int32_t ldv,
                                  int32_t t, uint64_t pos, uint64_t seq, uint64_t block_table, int32_t n_seqs, int32_t max_pages,
                                  const dsuf_rope* rope, uint64_t q, int32_t ldq, int32_t q_heads, uint64_t q_out, int32_t ldqo,
                                  uint64_t k_out, int32_t ldko) {
    if (!ctx) return DSUF_E_BADARG;
    int rc = check_kv_cache(ctx, "kv_append", cache);
    if (rc) return rc;
    const int D = cache->head_dim;
    DSUF_REQUIRE(ctx, t >= 0 && n_seqs >= 0 && max_pages >= 1 && (long long)max_pages * cache->page_size <= 0x7fffffffll,
                 "kv_append: t, n_seqs >= 0, max_pages >= 1 and fewer than 2^31 positions");
    DSUF_REQUIRE(ctx, seq || t <= n_seqs, "kv_append: without seq, token i is sequence i: t (%d) must be at most n_seqs (%d)", t, n_seqs);
    DSUF_REQUIRE(ctx, q_heads >= 0 && q_heads <= 4096, "kv_append: q_heads (%d) must be in 0..4096", q_heads);
    DSUF_REQUIRE(ctx, ldk >= cache->kv_heads * D && ldk % 8 == 0 && ldv >= cache->kv_heads * D && ldv % 8 == 0,
                 "kv_append: ldk and ldv must be multiples of 8 and hold kv_heads * head_dim elements");
    DSUF_REQUIRE(ctx, !q_heads || (ldq >= q_heads * D && ldq % 8 == 0 && ldqo >= q_heads * D && ldqo % 8 == 0),
                 "kv_append: ldq and ldqo must be multiples of 8 and hold q_heads * head_dim elements");
    DSUF_REQUIRE(ctx, !k_out || (ldko >= cache->kv_heads * D && ldko % 8 == 0 && (k_out & 15) == 0),
                 "kv_append: k_out must be 16-byte aligned, ldko a multiple of 8 that holds kv_heads * head_dim elements");
    DSUF_REQUIRE(ctx, !rope || (rope->rot >= 16 && rope->rot % 16 == 0 && rope->off >= 0 && rope->off % 8 == 0 && rope->off <= D - rope->rot),
                 "kv_append: rope needs rot a multiple of 16, off a multiple of 8, off + rot <= head_dim");
    DSUF_REQUIRE(ctx, !rope || (rope->cos && rope->sin && (rope->cos & 15) == 0 && (rope->sin & 15) == 0 && rope->positions >= 1),
                 "kv_append: rope tables must be 16-byte aligned and hold at least one position");
    if (t == 0) return DSUF_OK;
    DSUF_REQUIRE(ctx, k && v && pos && block_table && (k & 15) == 0 && (v & 15) == 0 && (pos & 3) == 0 && (seq & 3) == 0 && (block_table & 3) == 0,
                 "kv_append: null or misaligned pointer (k, v 16 bytes, indexes 4)");
    DSUF_REQUIRE(ctx, !q_heads || (q && q_out && (q & 15) == 0 && (q_out & 15) == 0), "kv_append: q and q_out must be 16-byte aligned");
    const long long wq = (long long)q_heads * D, wk = (long long)cache->kv_heads * D;
    DSUF_REQUIRE(ctx, !q_heads || ((rows_in_place(q_out, ldqo, q, ldq, t) || !rows_overlap(q_out, ldqo, wq, q, ldq, wq, t)) &&
                 !rows_overlap(q_out, ldqo, wq, k, ldk, wk, t) && !rows_overlap(q_out, ldqo, wq, v, ldv, wk, t)),
                 "kv_append: q_out must be q itself, row for row, or share no memory with q, k and v");
    DSUF_REQUIRE(ctx, !k_out || ((rows_in_place(k_out, ldko, k, ldk, t) || !rows_overlap(k_out, ldko, wk, k, ldk, wk, t)) && !rows_overlap(k_out, ldko, wk, v, ldv, wk, t) &&
                 (!q_heads || (!rows_overlap(k_out, ldko, wk, q, ldq, wq, t) && !rows_overlap(k_out, ldko, wk, q_out, ldqo, wq, t)))),
                 "kv_append: k_out must be k itself, row for row, or share no memory with k, v, q and q_out");
    DSUF_REQUIRE_DEVICE(ctx, "kv_append");
    AppendArgs a;
    memset(&a, 0, sizeof(a));
    a.q = (const bf16*)q; a.k = (const bf16*)k; a.v = (const bf16*)v; a.q_out = (bf16*)q_out; a.k_out = (bf16*)k_out;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldqo = ldqo; a.ldko = ldko;
    a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.n_seqs = n_seqs; a.max_pages = max_pages; a.n_pages = cache->n_pages;
    a.page_shift = __builtin_ctz((unsigned)cache->page_size);
    a.pos = (const int*)pos; a.seq = (const int*)seq; a.table = (const int*)block_table;
    a.ck = (uint8_t*)cache->k; a.cv = (uint8_t*)cache->v;
    a.k_scale = (const float*)cache->k_scale; a.v_scale = (const float*)cache->v_scale;
    a.page_stride = cache->page_stride;
    if (rope) {
        a.cos = (const float*)rope->cos; a.sin = (const float*)rope->sin;
        a.rope_rows = rope->positions; a.rot = rope->rot; a.off = rope->off;
    }
    a.status = ctx->dev_status;
    // few tokens: several CTAs share a token's heads, so that its loads are not queued behind one another in one CTA
    const int groups = ((q_heads + 2 * cache->kv_heads) * (D / 8) + AP_THREADS - 1) / AP_THREADS;
    int share = (2 * ctx->sm_count + t - 1) / t;
    if (share > groups) share = groups;
    void (*kern)(AppendArgs);
    const bool fp8 = cache->dtype == DSUF_KV_E4M3, half = rope && rope->half;
    if (D == 64) kern = fp8 ? (half ? kv_append_kernel<64, true, true> : kv_append_kernel<64, true, false>)
                            : (half ? kv_append_kernel<64, false, true> : kv_append_kernel<64, false, false>);
    else kern = fp8 ? (half ? kv_append_kernel<128, true, true> : kv_append_kernel<128, true, false>)
                    : (half ? kv_append_kernel<128, false, true> : kv_append_kernel<128, false, false>);
    return launch(ctx, (cudaStream_t)stream, kern, dim3(t, share), dim3(AP_THREADS), 0, a);
}
