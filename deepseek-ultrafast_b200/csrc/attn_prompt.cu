// Causal attention over packed prompts (dsuf_attn_prompt): grouped heads, ragged lengths, sliding window, bf16.
//
// out_i = sum_{j <= i} exp(scale <q_i, k_j> - top_i) v_j / sum: 4 D flops per visible pair against 2 D (2 hq + 2 hkv) bytes per
// token, so it is bound by the tensor cores and, as tightly, by the exponential unit (a 128 x 128 tile of scores costs 2 x 512 tensor
// cycles at D = 128 and 1024 cycles of 16 exponentials per clock and SM).
//
// One persistent CTA per SM works on two 128-row query tiles at a time that share their keys and values; the tiles of a (sequence,
// kv head) are numbered block * group + head-in-group and paired in that order, so a pair is almost always two heads of the same block
// and has one causal boundary (an odd group pairs the last head of a block with the first of the next).  Roles:
//   warps 0-3, 4-7   softmax of tile 0 / 1: a thread owns a row; scores from tensor memory, p back to tensor memory
//   warp 8           TMA: query tiles, and a ring of key / value tiles (K0 V0 K1 V1 ...)
//   warp 9, 10       tcgen05.mma of tile 0 / 1: S_t = Q_t K^T (operands in shared memory), O_t += P_t V (P in tensor memory, V as it
//                    lies, tokens by columns, through the MN-major operand form)
// The tensor core works on one tile while the other tile's softmax runs; S of step j + 1 is issued behind PV of step j, so its
// completion also says that the output may be rescaled.  The steps of successive pairs form one stream: the next pair's first scores are
// issued before the last output is stored.  The two issuing warps take strict turns (P0 V, S0, P1 V, S1): issuing blocks while the tensor
// core's short queue is full, so the barrier waits of one tile (100 cycles and more each, even when met) have to pass while the
// other's products are issued; without turns the tiles fall into step, and both softmaxes share the exponential unit and then both wait.
// (8192 tokens, 56 / 8 heads of 128: one issuing warp 867 us, two without turns 1022, two with turns 778; now 755 to 795 from one GPU to another,
// 1270 TFLOP/s of visible pairs at best; in a capture of 4096 tokens the tensor pipe was 54 % and the exponential unit 55 % busy.)
// Tensor memory (512 columns): S0 S1 (128 fp32 columns each; P_t overwrites the first 64 of S_t as packed bf16), O0 O1 (D each).
// The reference point of a row is the largest of 16 or 32 scores of its first tile and only moves when a tile's weights add up to more than 2^24 (exact: the
// sum and the output share the reference, and bf16's and fp32's precision does not depend on the magnitude), so usual tiles need no maximum at
// all.  Sums, statistics and outputs are fp32.  p is rounded once to bf16 as operand: the outputs' error against 64 bits is then 0.0020 of their norm, where
// that of their own rounding is 0.0016.  A second bf16 number for what the rounding leaves, as decode attention has it, would take 64 registers more
// of a softmax thread that has none left, twice the stores of p and half as many products again (here the tensor core is as tight as anything).
//
// Pairs are ordered from the longest rows to the shortest, those of all sequences together, and dealt to the CTAs back and forth, which
// leaves the CTAs within 1 or 2 % of one another (9 prompts of 900 to 2600 tokens: 332 us; sequence after sequence 8 % apart and 342; one of 2048 69 instead of 74).  Values behind a sequence's end inside its last tile belong to another sequence (or nobody) and are
// zeroed in shared memory before use: p is 0 there, but 0 x NaN is not.
#include "internal.h"

namespace dsuf {

constexpr int KID_PROMPT = 9;
constexpr int PA_THREADS = 352;
constexpr int PA_BM = 128;
constexpr float PA_UNSET = -3.4028234663852886e38f;     // no finite score is below it
constexpr float PA_TRIGGER = 16777216.f;
constexpr float PA_FAR = 268435456.f;   // beyond this a reference's own rounding is an exponent of more than 8

template <int D>
struct PromptShape {
    static constexpr int BOXES = D / 64;                       // 128-byte wide operand boxes of a tile
    static constexpr int TILE = PA_BM * D * 2;                 // bytes of a query, key or value tile
    static constexpr int STAGES = D == 128 ? 4 : 8;            // ring of key / value tiles
    static constexpr int OUT = 32 * 128;                       // a warp's staging for its output: 32 rows of 64 columns
    static constexpr int SMEM = 2 * TILE + STAGES * TILE + 8 * OUT + 1024;
};

struct PromptArgs {
    CUtensorMap tm_q, tm_k, tm_v;
    const bf16 *q, *k, *v;          // the same rows, for prompt_repair, which is seldom needed
    int ldq, ldk, ldv;
    bf16* out;
    float* lse;
    int ldo, t, q_heads, kv_heads, group, n_seqs, window;
    const int* cu;
    float scale_log2;
    DevStatus* status;
};

// kind::f16, fp32 accumulator, bf16 operands, M = 128; bit 16: B is MN-major.
DSUF_DEV constexpr uint32_t pa_idesc(int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n / 8) << 17) | ((uint32_t)(128 / 16) << 24);
}
DSUF_DEV void pa_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        "  .reg .pred keep_d;\n"
        "  setp.ne.u32 keep_d, %4, 0;\n"
        "  tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, keep_d;\n"
        "}\n"
        :
        : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
DSUF_DEV void pa_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        "  .reg .pred keep_d;\n"
        "  setp.ne.u32 keep_d, %4, 0;\n"
        "  tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, keep_d;\n"
        "}\n"
        :
        : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
#define PA_R4(v, i) "r"(v[i]), "r"(v[(i) + 1]), "r"(v[(i) + 2]), "r"(v[(i) + 3])
#define PA_R16(v, i) PA_R4(v, i), PA_R4(v, (i) + 4), PA_R4(v, (i) + 8), PA_R4(v, (i) + 12)
DSUF_DEV void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        :
        : PA_R16(v, 0), "r"(taddr)
        : "memory");
}
DSUF_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" : : : "memory"); }
DSUF_DEV float pa_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
DSUF_DEV uint32_t pa_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// A query tile: rows [qb * 128, ..) of the sequence, query head, key tiles [lo, hi) (hi = 0: no tile).
struct PromptTile {
    int qb, head, lo, hi;
    DSUF_DEV bool active(int j) const { return j >= lo && j < hi; }
};
// A pair of them, of sequence rows start .. start + len - 1; together they need the key tiles [jlo, jhi).
struct PromptPair {
    int start, len, kvh;
    PromptTile t0, t1;
    int jlo, jhi;
    bool ok;
    DSUF_DEV PromptTile tile(int t) const {     // (selects, so that the pair stays in registers)
        PromptTile r;
        r.qb = t ? t1.qb : t0.qb;
        r.head = t ? t1.head : t0.head;
        r.lo = t ? t1.lo : t0.lo;
        r.hi = t ? t1.hi : t0.hi;
        return r;
    }
};

// Walks the pairs of one CTA: row r of the deal takes index r * grid + c, or counted from the other end in odd rows.  The indexes go by level, the number
// of key tiles up to a pair's diagonal, from the highest down, and inside a level by sequence.  Of a sequence of T blocks of 128 rows, blocks h - 1 and
// before have h group query tiles, so the pairs of level h are those from (h - 1) group / 2 to h group / 2 (T group / 2 rounded up, for the last): how many
// pairs a level has follows from the numbers of sequences with T > h and T = h.  A whole warp calls next() together: its lanes look at 32 sequences at a time.
struct PromptWalk {
    const PromptArgs& a;
    int row = 0, seq = 0, level = 0;      // seq: first of the 32 sequences looked at
    long long before = 0;                 // pairs of the levels above, and of the sequences below it in this one
    DSUF_DEV explicit PromptWalk(const PromptArgs& a_) : a(a_) {
        for (int s = 0; s < a.n_seqs; s += 32) {
            int start, len;
            bounds(s + (threadIdx.x & 31), start, len);
            level = max(level, (len + PA_BM - 1) / PA_BM);
        }
        level = __reduce_max_sync(0xffffffffu, level);
    }
    DSUF_DEV void bounds(int s, int& start, int& len) const {
        start = len = 0;
        if (s < a.n_seqs) {
            start = min(max(__ldg(a.cu + s), 0), a.t);
            len = max(min(max(__ldg(a.cu + s + 1), 0), a.t) - start, 0);
        }
    }
    DSUF_DEV PromptTile tile(int it, int tiles, int kvh) const {
        PromptTile t;
        t.qb = it / a.group;
        t.head = kvh * a.group + it % a.group;
        t.hi = it < tiles ? t.qb + 1 : 0;
        t.lo = it < tiles && a.window > 0 ? max(0, t.qb * PA_BM - a.window + 1) / PA_BM : 0;
        return t;
    }
    DSUF_DEV PromptPair next() {
        const int lane = threadIdx.x & 31;
        const unsigned below = (2u << lane) - 1u;      // the lanes up to this one
        PromptPair p;
        p.ok = false;
        const long long x = (long long)row * gridDim.x + ((row & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        ++row;
        int start = 0, len = 0;
        for (bool load = true; level > 0; load = a.n_seqs > 32) {
            if (load) bounds(seq + lane, start, len);
            const int blocks = (len + PA_BM - 1) / PA_BM;
            const unsigned higher = __ballot_sync(0xffffffffu, blocks > level), here = __ballot_sync(0xffffffffu, blocks == level);
            const int first = (level - 1) * a.group / 2, full = level * a.group / 2 - first, last = (level * a.group + 1) / 2 - first;      // pairs per kv head
            const int all = (__popc(higher) * full + __popc(here) * last) * a.kv_heads;
            if (x < before + all) {
                const int upto = (__popc(higher & below) * full + __popc(here & below) * last) * a.kv_heads;
                const int owner = __ffs(__ballot_sync(0xffffffffu, before + upto > x)) - 1;
                const int mine = (blocks > level ? full : blocks == level ? last : 0) * a.kv_heads;
                const int local = (int)(x - before) - __shfl_sync(0xffffffffu, upto - mine, owner);
                p.start = __shfl_sync(0xffffffffu, start, owner);
                p.len = __shfl_sync(0xffffffffu, len, owner);
                const int tiles = ((p.len + PA_BM - 1) / PA_BM) * a.group;
                const int pair = first + local / a.kv_heads;
                p.kvh = local % a.kv_heads;
                p.t0 = tile(2 * pair, tiles, p.kvh);
                p.t1 = tile(2 * pair + 1, tiles, p.kvh);
                p.jlo = p.t0.lo;                              // (the second tile's rows are the same or later ones)
                p.jhi = max(p.t0.hi, p.t1.hi);
                p.ok = true;
                return p;
            }
            before += all;
            seq += 32;
            if (seq >= a.n_seqs) {
                seq = 0;
                --level;
            }
        }
        return p;
    }
};

// One row's 128 scores in chunks of 32 columns, the next chunk's load under way while `f(chunk, values)` works on one.
template <typename F>
DSUF_DEV void pa_chunks(uint32_t tS, F f) {
    float s[2][32];
    tmem_ld_issue<32>(tS, s[0]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        tmem_wait_ld();
        if (c < 3) tmem_ld_issue<32>(tS + (c + 1) * 32, s[(c + 1) & 1]);
        f(c, s[c & 1]);
    }
}
DSUF_DEV float pa_total(unsigned long long two) {
    float x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(two));
    return x + y;
}
DSUF_DEV bool pa_far(float ref) { return fabsf(ref) > PA_FAR && ref > PA_UNSET; }
DSUF_DEV bool pa_seen(int col, int upper, int lower) { return col <= upper && col > lower; }
// p = 2^(s sl2 - ref) of a row, packed to bf16 in w, and their sum.  MASK 0: all columns are visible, 1: those up to `upper`, 2: those above
// `lower` as well, 3: the same, and the product s sl2 is rounded as a far reference was.
template <int MASK>
DSUF_DEV float pa_weights(uint32_t tS, float sl2, float ref, int upper, int lower, uint32_t* w) {
    const unsigned long long scale2 = pack_f32x2(sl2, sl2), ref2 = pack_f32x2(-ref, -ref);
    unsigned long long sum2 = pack_f32x2(0.f, 0.f);
    pa_chunks(tS, [&](int c, float* s) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            unsigned long long v;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(pack_f32x2(s[e], s[e + 1])), "l"(scale2), "l"(ref2));
            float x, y;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
            if (MASK == 3 && pa_far(ref)) {
                x = __fsub_rn(__fmul_rn(s[e], sl2), ref);
                y = __fsub_rn(__fmul_rn(s[e + 1], sl2), ref);
            }
            if constexpr (MASK > 0) {
                const int col = c * 32 + e;
                x = pa_seen(col, upper, MASK > 1 ? lower : -1) ? x : -INFINITY;
                y = pa_seen(col + 1, upper, MASK > 1 ? lower : -1) ? y : -INFINITY;
            }
            x = pa_exp2(x);
            y = pa_exp2(y);
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum2) : "l"(pack_f32x2(x, y)));
            w[c * 16 + e / 2] = pa_pack(x, y);
        }
    });
    return pa_total(sum2);
}

// Which of 32 consecutive bf16 at `p` (16-byte aligned) are not finite, and which are NaN, a bit for each.
DSUF_DEV void pa_odd32(const bf16* p, uint32_t& odd, uint32_t& nan) {
    odd = nan = 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const uint4 x = reinterpret_cast<const uint4*>(p)[v];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t m = (w[e / 2] >> (16 * (e & 1))) & 0x7fffu;
            odd |= (m >= 0x7f80u ? 1u : 0u) << (v * 8 + e);
            nan |= (m > 0x7f80u ? 1u : 0u) << (v * 8 + e);
        }
    }
}

DSUF_DEV void pa_mma_sync(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// In the tiles that the diagonal or the window cuts, the tensor core multiplies hidden values with p = 0, and 0 x infinity is NaN.  A softmax warp that
// has met outputs that are not finite comes here when the CTA is done otherwise (nobody waits for it then, however long its rows are), walks its tiles
// again, and where an output is NaN, a value of its column that is hidden from the row is not finite in those tiles, and no visible one there is NaN, the
// output is computed again from the row's visible keys alone: a row per lane and 32 columns at a time (8192 tokens, 56 / 8 heads of 128, one NaN in the
// last tile: 2.0 ms more; a row of NaN in every head: 7.8).
constexpr int PA_KEYS = 16;
constexpr int PA_REPAIR = 32 * (PA_KEYS + 1) * 4 + PA_KEYS * 32 * 4;     // bytes of shared memory of a warp: scores and values
template <int D>
__device__ __noinline__ void prompt_repair(const PromptArgs& a) {
    extern __shared__ uint8_t smem_raw[];      // (its address and the tile worked out here: as arguments they cost the caller registers, and 2 % of its time)
    const int t = threadIdx.x >> 7;
    float* scores = reinterpret_cast<float*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u) + (threadIdx.x >> 5) * PA_REPAIR);
    static_assert(PA_REPAIR % 16 == 0 && (32 * (PA_KEYS + 1) * 4) % 16 == 0 && 8 * PA_REPAIR <= PromptShape<D>::SMEM - 1024, "scores and values fit");
    float* values = scores + 32 * (PA_KEYS + 1);
    const int lane = threadIdx.x & 31, first = ((threadIdx.x >> 5) & 3) * 32;
    PromptWalk walk(a);
    for (;;) {
        const PromptPair p = walk.next();
        if (!p.ok) break;
        const PromptTile q = p.tile(t);
        const int tile0 = q.qb * PA_BM, row0 = tile0 + first, i = row0 + lane;
        if (q.hi == 0 || row0 >= p.len) continue;
        const bool live = i < p.len;
        const int from = a.window > 0 ? max(0, i - a.window + 1) : 0;
        const int end = min(p.len, tile0 + PA_BM);                                    // of the diagonal tile
        const int lower = a.window > 0 ? min(tile0, row0 + 32 - a.window) : 0;        // of the keys that the window hides from one of the rows
        bf16* out = a.out + (size_t)(p.start + (live ? i : row0)) * a.ldo + (size_t)q.head * D;
        const bf16* kb = a.k + (size_t)p.start * a.ldk + (size_t)p.kvh * D;
        const bf16* vb = a.v + (size_t)p.start * a.ldv + (size_t)p.kvh * D;
        for (int c = 0; c < D; c += 32) {
            uint32_t nan, hidden = 0, seen = 0;
            pa_odd32(out + c, hidden, nan);
            if (!live) nan = 0;
            if (!__any_sync(0xffffffffu, nan != 0)) continue;
            hidden = 0;
            for (int j0 = q.lo * PA_BM; j0 < end; j0 += 32) {
                if (j0 >= lower && j0 < tile0) j0 = tile0;                            // (uncut tiles hide nothing)
                uint32_t odd_here = 0, nan_here = 0;
                if (j0 + lane < end) pa_odd32(vb + (size_t)(j0 + lane) * a.ldv + c, odd_here, nan_here);
                if (!__any_sync(0xffffffffu, odd_here != 0)) continue;
                for (int m = 0; m < 32; ++m) {
                    const uint32_t o = __shfl_sync(0xffffffffu, odd_here, m), n = __shfl_sync(0xffffffffu, nan_here, m);
                    if (j0 + m >= from && j0 + m <= i) seen |= n;
                    else hidden |= o;
                }
            }
            const uint32_t wrong = nan & hidden & ~seen;
            if (!__any_sync(0xffffffffu, wrong != 0)) continue;
            // scores of 32 rows and 16 keys by mma.sync, through shared memory to a row per lane.  Its sums over the head's columns may take these in any order:
            // of each 32 a lane has 8 beside each other, as the operands of two steps.
            uint4 qf[4][D / 32];                     // rows lane / 4 + 8 r
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int v = 0; v < D / 32; ++v)
                    qf[r][v] = reinterpret_cast<const uint4*>(a.q + (size_t)(p.start + min(row0 + r * 8 + lane / 4, p.len - 1)) * a.ldq + (size_t)q.head * D)[v * 4 + lane % 4];
            float o[32], top = PA_UNSET, sum = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
            const int j_from = __reduce_min_sync(0xffffffffu, wrong ? from : 0x7fffffff), j_to = __reduce_max_sync(0xffffffffu, wrong ? i : -1);
            for (int j0 = j_from; j0 <= j_to; j0 += PA_KEYS) {
                uint4 y[PA_KEYS / 8];
#pragma unroll
                for (int v = 0; v < PA_KEYS / 8; ++v) y[v] = __ldg(reinterpret_cast<const uint4*>(vb + (size_t)min(j0 + v * 8 + lane / 4, j_to) * a.ldv + c) + lane % 4);
                __syncwarp();                        // (the last scores and values have been read)
#pragma unroll
                for (int n = 0; n < PA_KEYS / 8; ++n) {
                    const uint4* kr = reinterpret_cast<const uint4*>(kb + (size_t)min(j0 + n * 8 + lane / 4, j_to) * a.ldk) + lane % 4;
                    float s[2][4] = {};
#pragma unroll
                    for (int v = 0; v < D / 32; ++v) {
                        const uint4 x = __ldg(kr + v * 4);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            pa_mma_sync(s[m], qf[2 * m][v].x, qf[2 * m + 1][v].x, qf[2 * m][v].y, qf[2 * m + 1][v].y, x.x, x.y);
                            pa_mma_sync(s[m], qf[2 * m][v].z, qf[2 * m + 1][v].z, qf[2 * m][v].w, qf[2 * m + 1][v].w, x.z, x.w);
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) scores[(m * 16 + (e >> 1) * 8 + lane / 4) * (PA_KEYS + 1) + n * 8 + lane % 4 * 2 + (e & 1)] = s[m][e];
                }
#pragma unroll
                for (int v = 0; v < PA_KEYS / 8; ++v) {
                    const uint32_t w[4] = {y[v].x, y[v].y, y[v].z, y[v].w};
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
                        *reinterpret_cast<float4*>(values + (v * 32 + lane) * 8 + 2 * e) = make_float4(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u),
                                                                                                   __uint_as_float(w[e + 1] << 16), __uint_as_float(w[e + 1] & 0xffff0000u));
                }
                __syncwarp();
#pragma unroll 4
                for (int m = 0; m < PA_KEYS; ++m) {
                    const float s = scores[lane * (PA_KEYS + 1) + m] * a.scale_log2;
                    if (!wrong || j0 + m < from || j0 + m > i) continue;
                    if (s > top) {
                        const float by = pa_exp2(top - s);
                        top = s;
                        sum *= by;
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= by;
                    }
                    const float w = pa_exp2(s - top);
                    sum += w;
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = fmaf(w, values[m * 32 + e], o[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if ((wrong >> e) & 1) out[c + e] = __float2bfloat16(sum == 0.f ? 0.f : o[e] / sum);
        }
    }
}

// WINDOW: with a sliding window (a kernel of its own: what only windows need costs the other 4 % of its time).
template <int D, bool WINDOW>
__global__ void __launch_bounds__(PA_THREADS, 1) attn_prompt_kernel(const __grid_constant__ PromptArgs a) {
    using S = PromptShape<D>;
    constexpr int BOX = PA_BM * 128;                 // bytes of one box
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* ring = base + 2 * S::TILE;
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], kv_full[S::STAGES], kv_empty[S::STAGES], s_full[2], p_full[2], o_full[2], drained[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_odd[8];         // softmax warps that have met outputs which are not finite
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    bool dead = false;

    if (warp == 8) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    if (tid < 8) s_odd[tid] = 0;
    if (tid == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_full[t], 1);
            mbar_init(&drained[t], 1);
        }
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&kv_empty[s], 2);
        }
        mbar_fence_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = s_tmem;
    pdl_wait();
    pdl_launch_dependents();
    PromptWalk walk(a);

    if (warp == 8) {
        // ---------------- producer ----------------
        if (lane == 0) {
            prefetch_tmap(&a.tm_q);
            prefetch_tmap(&a.tm_k);
            prefetch_tmap(&a.tm_v);
        }
        int st = 0;
        uint32_t ph = 0, qn[2] = {0, 0}, copied = 0, qcopied[2] = {0, 0};
        long long n = 0;
        auto kv = [&](const PromptPair& p, const CUtensorMap* map, int j) {
            if (n >= S::STAGES && !dead && !mbar_wait(&kv_empty[st], ph ^ 1, a.status, KID_PROMPT, 1)) dead = true;
            if (warp_elect() && !dead) {        // (else nothing is copied any more, and what has been is awaited below)
                ++copied;
                mbar_expect_tx(&kv_full[st], S::TILE);
#pragma unroll
                for (int b = 0; b < S::BOXES; ++b)
                    tma_2d_nh(ring + st * S::TILE + b * BOX, map, p.kvh * D + b * 64, p.start + j * PA_BM, &kv_full[st]);
            }
            __syncwarp();
            ++n;
            if (++st == S::STAGES) { st = 0; ph ^= 1; }
        };
        for (;;) {
            const PromptPair p = walk.next();
            if (!p.ok) break;
            kv(p, &a.tm_k, p.jlo);   // ahead of the queries: their buffers become free later than the ring's
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const PromptTile q = t ? p.t1 : p.t0;
                if (q.hi == 0) continue;
                if (qn[t] > 0 && !dead && !mbar_wait(&q_empty[t], (qn[t] - 1) & 1, a.status, KID_PROMPT, 2)) dead = true;
                if (warp_elect() && !dead) {
                    ++qcopied[t];
                    mbar_expect_tx(&q_full[t], S::TILE);
#pragma unroll
                    for (int b = 0; b < S::BOXES; ++b)
                        tma_2d_nh(base + t * S::TILE + b * BOX, &a.tm_q, q.head * D + b * 64, p.start + q.qb * PA_BM, &q_full[t]);
                }
                __syncwarp();
                ++qn[t];
            }
            for (int j = p.jlo; j < p.jhi; ++j) {
                if (j > p.jlo) kv(p, &a.tm_k, j);
                kv(p, &a.tm_v, j);
            }
        }
        // no CTA ends with copies on their way: the last one into each stage, and of each tile's queries
        copied = __reduce_add_sync(0xffffffffu, copied);
        for (uint32_t s = 0; s < min(copied, (uint32_t)S::STAGES); ++s) mbar_wait(&kv_full[s], ((copied - 1 - s) / S::STAGES) & 1, a.status, KID_PROMPT, 8);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t of = __reduce_add_sync(0xffffffffu, qcopied[t]);
            if (of > 0) mbar_wait(&q_full[t], (of - 1) & 1, a.status, KID_PROMPT, 9);
        }
    } else if (warp >= 9) {
        // ---------------- tensor core issuer of tile t ----------------
        const int t = warp - 9;
        const uint32_t tmS = warp_uniform(tm + t * 128), tmO = warp_uniform(tm + 256 + t * D);
        // operand descriptors: the address is in the low word, so steps are 32-bit additions
        const uint64_t kmajor = tc_smem_desc(base, 16, 1024, TC_SWIZZLE_128B);
        const uint32_t desc_hi = warp_uniform((uint32_t)(kmajor >> 32)), q_lo = warp_uniform((uint32_t)kmajor + ((t * S::TILE) >> 4));
        const uint32_t ring_lo = warp_uniform((uint32_t)tc_smem_desc(ring, 16, 1024, TC_SWIZZLE_128B));
        const uint32_t ring_lo_v = warp_uniform((uint32_t)tc_smem_desc(ring, BOX, 1024, TC_SWIZZLE_128B));   // column chunks of 64 a box apart, 8 tokens 1024 bytes
        int st = 0;
        uint32_t ph = 0, qn = 0, pn = 0;
        auto wait_kv = [&]() {
            if (!dead && !mbar_wait(&kv_full[st], ph, a.status, KID_PROMPT, 3)) dead = true;
            tc_fence_after();
        };
        // the stage is free once what this warp has issued is done, and the other tile's warp says the same
        auto release_kv = [&](int stage) {
            if (warp_elect()) tc_commit(&kv_empty[stage]);
            __syncwarp();
        };
        auto advance = [&]() {
            if (++st == S::STAGES) { st = 0; ph ^= 1; }
        };
        auto desc = [&](uint32_t lo) { return ((uint64_t)desc_hi << 32) | lo; };
        // the turn, handed to and fro on two named barriers; both warps walk the same steps, so every arrival is awaited
        auto take_turn = [&]() { named_bar_sync(2 + t, 64); };
        auto pass_turn = [&]() { named_bar_arrive(2 + (t ^ 1), 64); };
        auto wait_q = [&](const PromptTile& q, int j) {
            if (j == q.lo) {
                if (!dead && !mbar_wait(&q_full[t], qn & 1, a.status, KID_PROMPT, 4)) dead = true;
                ++qn;
                tc_fence_after();
            }
        };
        auto scores = [&](const PromptTile& q, int j, uint32_t k_lo) {
            const bool last = j == q.hi - 1;
            if (warp_elect()) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const uint32_t off = (uint32_t)((c >> 2) * BOX + (c & 3) * 32) >> 4;
                    pa_mma_ss(tmS, desc(q_lo + off), desc(k_lo + off), pa_idesc(128, false), c != 0);
                }
                tc_commit(&s_full[t]);
                if (last) tc_commit(&q_empty[t]);
            }
            __syncwarp();
        };
        if (t == 1) pass_turn();     // tile 0 begins
        PromptPair cur = walk.next();
        PromptTile mine = cur.tile(t);
        if (cur.ok) {
            wait_kv();
            const uint32_t k_lo = warp_uniform(ring_lo + ((st * S::TILE) >> 4));
            const bool go = mine.active(cur.jlo);
            if (go) wait_q(mine, cur.jlo);
            take_turn();
            if (go) scores(mine, cur.jlo, k_lo);
            pass_turn();
            release_kv(st);
            advance();
        }
        while (cur.ok) {
            PromptPair nxt = cur;
            PromptTile then = mine;      // what the next step's scores belong to
            for (int j = cur.jlo; j < cur.jhi; ++j) {
                const bool last = j + 1 == cur.jhi;
                if (last) {
                    nxt = walk.next();
                    then = nxt.tile(t);
                }
                const bool more = nxt.ok;
                const int nj = last ? nxt.jlo : j + 1;
                const bool here = mine.active(j), next = more && then.active(nj);
                wait_kv();
                const int vst = st;
                advance();
                const int behind = cur.len - j * PA_BM;      // rows of this tile inside the sequence
                if (here && behind < PA_BM) {
                    // (both tiles' warps may write these zeros, the second while the first one's product reads them)
                    for (int i = lane; i < (PA_BM - behind) * 8 * S::BOXES; i += 32) {
                        const int b = i / ((PA_BM - behind) * 8), r = i % ((PA_BM - behind) * 8);
                        *reinterpret_cast<uint4*>(ring + vst * S::TILE + b * BOX + behind * 128 + r * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                    __syncwarp();
                }
                const uint32_t v_lo = warp_uniform(ring_lo_v + ((vst * S::TILE) >> 4)), k_lo = warp_uniform(ring_lo + ((st * S::TILE) >> 4));
                const bool first = j == mine.lo, end = j == mine.hi - 1;
                if (more) wait_kv();
                if (next) wait_q(then, nj);
                if (here) {
                    if (!dead && !mbar_wait(&p_full[t], pn & 1, a.status, KID_PROMPT, 5)) dead = true;
                    ++pn;
                    tc_fence_after();
                }
                take_turn();
                if (here) {
                    if (warp_elect()) {
#pragma unroll
                        for (int c = 0; c < PA_BM / 16; ++c) pa_mma_ts(tmO, tmS + c * 8, desc(v_lo + c * 128), pa_idesc(D, true), c != 0 || !first);
                        if (end) tc_commit(&o_full[t]);
                    }
                    __syncwarp();
                }
                if (next) scores(then, nj, k_lo);
                pass_turn();
                release_kv(vst);
                if (more) {
                    release_kv(st);
                    advance();
                }
            }
            cur = nxt;
            mine = then;
        }
        if (t == 0) take_turn();     // (the last turn that tile 1 has passed on)
        // nor with products on their way, whose operands and results the CTA's memory holds
        if (warp_elect()) tc_commit(&drained[t]);
        __syncwarp();
        mbar_wait(&drained[t], 0, a.status, KID_PROMPT, 10);
    } else {
        // ---------------- softmax: tile t, one row per thread ----------------
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tm + lanes + t * 128, tO = tm + lanes + 256 + t * D;
        const int r = (warp & 3) * 32 + lane;        // row inside the tile
        const float sl2 = a.scale_log2;
        uint8_t* stage = ring + S::STAGES * S::TILE + warp * S::OUT;
        uint32_t sn = 0, on = 0;
        PromptPair ahead = walk.next();
        for (;;) {
            const PromptPair p = ahead;
            if (!p.ok) break;
            const PromptTile q = p.tile(t);
            if (q.hi == 0) {
                ahead = walk.next();
                continue;
            }
            const int row = q.qb * PA_BM + r;
            float ref = PA_UNSET, sum = 0.f;
            for (int j = q.lo; j < q.hi; ++j) {
                if (!dead && !mbar_wait(&s_full[t], sn & 1, a.status, KID_PROMPT, 6)) dead = true;
                ++sn;
                tc_fence_after();
                const int upper = row - j * PA_BM;                                  // last visible column of the tile
                const int lower = WINDOW ? upper - a.window : -1;             // last column hidden by the window
                const bool windowed = WINDOW && q.qb * PA_BM + PA_BM - 1 - j * PA_BM >= a.window, diagonal = j == q.hi - 1;
                uint32_t w[64];
                if (WINDOW ? __any_sync(0xffffffffu, ref == PA_UNSET) : j == q.lo) {
                    // a row's first reference: the largest of some scores that it sees (of 16 without a window, where every row sees column 0: of 32, 1 % more
                    // of the kernel's time).  Of a tile that only the
                    // window cuts a row sees the last columns or none; where the diagonal cuts too, its own column.
                    const int at = !WINDOW || !windowed ? 0 : diagonal ? (warp & 3) * 32 : 96;
                    constexpr int FIRST = WINDOW ? 32 : 16;
                    float s[FIRST], top = -INFINITY;
                    tmem_ld<FIRST>(tS + at, s);
#pragma unroll
                    for (int e = 0; e < FIRST; ++e) top = fmaxf(top, pa_seen(at + e, upper, lower) ? s[e] : -INFINITY);
                    if (!WINDOW || ref == PA_UNSET) ref = fmaxf(top * sl2, PA_UNSET);
                }
                float part;
                if (WINDOW && windowed) part = pa_weights<2>(tS, sl2, ref, upper, lower, w);
                else if (diagonal) part = pa_weights<1>(tS, sl2, ref, upper, lower, w);
                else part = pa_weights<0>(tS, sl2, ref, upper, lower, w);
                const bool fine = part <= PA_TRIGGER && !pa_far(ref);
                if (!__all_sync(0xffffffffu, fine)) {
                    // (seldom, or NaN, or scores of 2^28 and more) the reference moves up to the tile's largest score where that is larger; so do the sum and the output, which is
                    // complete: this step's scores were issued behind the last step's product
                    float top = PA_UNSET;
#pragma unroll 1
                    for (int c = 0; c < 128; c += 16) {
                        float s[16];
                        tmem_ld<16>(tS + c, s);
#pragma unroll
                        for (int e = 0; e < 16; ++e) top = fmaxf(top, pa_seen(c + e, upper, lower) ? __fmul_rn(s[e], sl2) : -INFINITY);
                    }
                    const float to = fine ? ref : fmaxf(ref, top);      // (a row's result does not depend on its neighbours)
                    const float by = pa_exp2(ref - to);
                    if (j > q.lo) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            float o[16];
                            tmem_ld<16>(tO + c, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= by;
                            tmem_st16(tO + c, reinterpret_cast<const uint32_t*>(o));
                        }
                    }
                    ref = to;
                    sum *= by;
                    part = pa_weights<3>(tS, sl2, ref, upper, lower, w);
                }
                sum += part;
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_st16(tS + c * 16, w + c * 16);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            ahead = walk.next();     // (while the last product is under way)
            if (!dead && !mbar_wait(&o_full[t], on & 1, a.status, KID_PROMPT, 7)) dead = true;
            ++on;
            tc_fence_after();
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const bool live = row < p.len;
            // through shared memory, so that a store instruction writes four rows of 128 bytes instead of 32 pieces of 16
            const int row0 = q.qb * PA_BM + (warp & 3) * 32;      // the warp's first row
            bf16* dst = a.out + (size_t)(p.start + row0) * a.ldo + (size_t)q.head * D;
            unsigned long long odd = pack_f32x2(0.f, 0.f);       // NaN once an output is not finite
#pragma unroll
            for (int c = 0; c < D; c += 64) {
                float o[64];
                tmem_ld_issue<32>(tO + c, o);
                tmem_ld_issue<32>(tO + c + 32, o + 32);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 64; e += 2)
                    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(odd) : "l"(pack_f32x2(o[e], o[e + 1])), "l"(pack_f32x2(0.f, 0.f)));
#pragma unroll
                for (int e = 0; e < 64; e += 8)
                    *reinterpret_cast<uint4*>(stage + lane * 128 + (((e / 8) ^ (lane & 7)) << 4)) =
                        make_uint4(pa_pack(o[e] * inv, o[e + 1] * inv), pa_pack(o[e + 2] * inv, o[e + 3] * inv),
                                   pa_pack(o[e + 4] * inv, o[e + 5] * inv), pa_pack(o[e + 6] * inv, o[e + 7] * inv));
                __syncwarp();
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const uint4*>(stage + (i * 4 + (lane >> 3)) * 128 + (((lane & 7) ^ ((i * 4 + (lane >> 3)) & 7)) << 4));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rr = i * 4 + (lane >> 3);
                    if (row0 + rr < p.len) *reinterpret_cast<uint4*>(dst + (size_t)rr * a.ldo + c + (lane & 7) * 8) = v[i];
                }
                __syncwarp();
            }
            if (live && !(pa_total(odd) == 0.f)) s_odd[warp] = 1;
            if (live && a.lse) a.lse[(size_t)(p.start + row) * a.q_heads + q.head] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tm, 512);
    if (warp < 8 && s_odd[warp]) prompt_repair<D>(a);
}

static int encode_heads(dsuf_ctx* ctx, CUtensorMap* tm, const void* base, long long width, long long ld, long long rows) {
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64u, (cuuint32_t)PA_BM};
    cuuint32_t es[2] = {1u, 1u};
    CUresult r = ctx->encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(ctx, DSUF_E_BADARG, "cuTensorMapEncodeTiled(attention) failed: %d", (int)r);
    return DSUF_OK;
}

template <int D, bool WINDOW>
static cudaError_t prompt_attr() { return cudaFuncSetAttribute(attn_prompt_kernel<D, WINDOW>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<D>::SMEM); }
int attn_prompt_setup(dsuf_ctx* ctx) {
    cudaError_t e = prompt_attr<64, false>();
    if (e == cudaSuccess) e = prompt_attr<64, true>();
    if (e == cudaSuccess) e = prompt_attr<128, false>();
    if (e == cudaSuccess) e = prompt_attr<128, true>();
    return e == cudaSuccess ? DSUF_OK : cuda_fail(ctx, e, "cudaFuncSetAttribute(attn_prompt)");
}

}  // namespace dsuf

using namespace dsuf;

extern "C" int32_t dsuf_attn_prompt(dsuf_ctx* ctx, void* stream, uint64_t q, int32_t ldq, uint64_t k, int32_t ldk, uint64_t v, int32_t ldv, int32_t t,
                                    int32_t q_heads, int32_t kv_heads, int32_t head_dim, uint64_t cu_seqlens, int32_t n_seqs, float scale,
                                    int32_t window, uint64_t out, int32_t ldo, uint64_t lse) {
    if (!ctx) return DSUF_E_BADARG;
    DSUF_REQUIRE(ctx, head_dim == 64 || head_dim == 128, "attn_prompt: head_dim (%d) must be 64 or 128", head_dim);
    DSUF_REQUIRE(ctx, kv_heads >= 1 && q_heads >= 1 && q_heads <= 4096 && q_heads % kv_heads == 0,
                 "attn_prompt: q_heads (%d) must be a multiple of kv_heads (%d), at most 4096", q_heads, kv_heads);
    // (a CTA looks for its next pair 32 sequences and a level at a time; with 2^18 sequences that is at most 296 levels x 8192 steps of about 1000 cycles,
    // as every other level has a pair, and stays inside the waits' limit of 4e9 cycles)
    DSUF_REQUIRE(ctx, t >= 0 && t <= 0x7fff0000 && n_seqs >= 0 && n_seqs <= 1 << 18, "attn_prompt: t must be in 0..2^31 - 65536 and n_seqs in 0..2^18");
    DSUF_REQUIRE(ctx, ldq >= q_heads * head_dim && ldq % 8 == 0 && ldo >= q_heads * head_dim && ldo % 8 == 0 && ldk >= kv_heads * head_dim && ldk % 8 == 0 &&
                 ldv >= kv_heads * head_dim && ldv % 8 == 0, "attn_prompt: row strides must be multiples of 8 and hold all heads");
    DSUF_REQUIRE(ctx, window >= 0 && scale > 0.f && scale - scale == 0.f, "attn_prompt: window must be >= 0, scale positive and finite");
    if (t == 0 || n_seqs == 0) return DSUF_OK;
    DSUF_REQUIRE(ctx, q && k && v && out && cu_seqlens && (q & 15) == 0 && (k & 15) == 0 && (v & 15) == 0 && (out & 15) == 0 && (cu_seqlens & 3) == 0 &&
                 (lse & 3) == 0, "attn_prompt: null or misaligned pointer (q, k, v, out 16 bytes, cu_seqlens and lse 4)");
    const long long wq = (long long)q_heads * head_dim, wk = (long long)kv_heads * head_dim;
    DSUF_REQUIRE(ctx, !rows_overlap(out, ldo, wq, q, ldq, wq, t) && !rows_overlap(out, ldo, wq, k, ldk, wk, t) && !rows_overlap(out, ldo, wq, v, ldv, wk, t),
                 "attn_prompt: out must not share memory with q, k or v");
    const long long lse_bytes = 4ll * t * q_heads;
    DSUF_REQUIRE(ctx, !lse || (!block_meets_rows(lse, lse_bytes, q, ldq, wq, t) && !block_meets_rows(lse, lse_bytes, k, ldk, wk, t) &&
                 !block_meets_rows(lse, lse_bytes, v, ldv, wk, t) && !block_meets_rows(lse, lse_bytes, out, ldo, wq, t)),
                 "attn_prompt: lse must share no memory with q, k, v and out");
    DSUF_REQUIRE_DEVICE(ctx, "attn_prompt");
    PromptArgs a;
    memset(&a, 0, sizeof(a));
    int rc = encode_heads(ctx, &a.tm_q, (const void*)q, wq, ldq, t);
    if (!rc) rc = encode_heads(ctx, &a.tm_k, (const void*)k, wk, ldk, t);
    if (!rc) rc = encode_heads(ctx, &a.tm_v, (const void*)v, wk, ldv, t);
    if (rc) return rc;
    a.out = (bf16*)out; a.lse = (float*)lse; a.ldo = ldo; a.t = t;
    a.q_heads = q_heads; a.kv_heads = kv_heads; a.group = q_heads / kv_heads; a.n_seqs = n_seqs; a.window = window;
    a.cu = (const int*)cu_seqlens;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.q = (const bf16*)q; a.k = (const bf16*)k; a.v = (const bf16*)v;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv;
    a.status = ctx->dev_status;
    // no more CTAs than pairs there can be (the lengths are only known on the device)
    const long long blocks = (long long)(t / PA_BM) + (t < n_seqs ? t : n_seqs);
    const long long cap = (blocks * a.group + 1) * kv_heads;
    const int grid = (int)(cap < ctx->sm_count ? cap : ctx->sm_count);
    const size_t smem = head_dim == 64 ? PromptShape<64>::SMEM : PromptShape<128>::SMEM;
    void (*kern)(PromptArgs) = head_dim == 64 ? (window ? attn_prompt_kernel<64, true> : attn_prompt_kernel<64, false>)
                                              : (window ? attn_prompt_kernel<128, true> : attn_prompt_kernel<128, false>);
    return launch(ctx, (cudaStream_t)stream, kern, dim3(grid), dim3(PA_THREADS), smem, a);
}
