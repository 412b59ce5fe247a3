// Attention of one new token per sequence over a paged key/value cache (dsuf_attn_decode): grouped heads, ragged lengths,
// sliding window, bf16 or e4m3 cache.
//
// out = sum_j exp(scale <q, k_j> - top) v_j / sum_j exp(scale <q, k_j> - top), one pass over the cache: HBM-bound, every
// visible key and value is read once and serves all query heads of its group (64 contexts of up to 8192 tokens, 56 / 8 heads of 128: 191 us = 6.0 TB/s,
// 0.92 of the measured copy bandwidth; one of 131071: 93 us, 0.88).  Groups of more than 16 heads read their keys once per 16 (32 contexts of 8192 over one kv head:
// 16 heads 37 us, 32 heads 50, 64 heads 76).
//
// Work split.  A piece is (sequence, kv head, block of 8 NT query heads); its keys are cut into units of 4 warps x CH tokens
// (CH tokens = 4 KB of keys), and all pieces' units, laid end to end, are dealt to the CTAs (two per SM) in equal contiguous
// ranges, computed on the device from seq_lens: ragged lengths balance to one unit, and nothing about the lengths has to be
// known on the host (a captured graph replays with new ones).  A piece inside one CTA is finished there; a piece cut by range
// ends leaves fp32 partials (output, reference point, sum) in the workspace and the CTA that arrives last adds them in CTA order,
// so the result does not depend on timing.  Where there are few units, segments of four of one piece are dealt instead of units (8 contexts
// of 1000 tokens, 56 / 8 heads of 128: 12.8 us instead of 14.5; one of 16000, one kv head: 14.0 instead of 24.6).  Where every piece is short (four
// units at most) and there is one for each CTA that the GPU holds, a warp takes whole pieces alone and writes them itself: no barrier and no other warp's part to add
// (56 / 8 heads of 128; 512 contexts of 128 tokens: 56 us instead of 68; 256 of 1 to 256: 37 instead of 61; 64 of 40: 7.6 instead of 10; with fewer pieces than
// CTAs it would lose: 256 pieces of 100 tokens 9.6 instead of 7.6).
//
// Inside a CTA every warp runs alone: a private ring of three stages (4 KB keys + 4 KB values each, cp.async, zero-filled
// outside the visible range so that stale values behind a sequence cannot reach the sums), no barrier until the end of a
// piece.  The loads run ahead over the piece boundaries.
//
// Products on mma.sync m16n8k16 with the TOKENS as the 16 rows (keys^T) and the query heads as the 8 columns: up to 8 heads of a
// group cost one column block where the usual orientation pads them to 16 rows (7 heads per kv head: half the instructions
// and accumulators).  S^T leaves the tensor core with a query head per thread column, which is also the layout of O^T = V^T P^T, so
// maxima, sums and rescaling need no shuffle; P^T is turned into an operand by two 8x8 register transposes (movmatrix).
// tcgen05 would add a shared-memory round trip for P for work that is a third of the memory time.
//
// Softmax: base-2 exponentials against a reference point that only moves when a score exceeds it by 2^15 (exact: the sum and the
// output share it); it is set 7 below the maximum so that p <= 2^15 and p's fp16 form keeps full precision down to 2^-21 of
// the largest.  Scores, sums and outputs are fp32.  As operand of the second product p is rounded to fp16
// (e4m3 cache), or split into two bf16 numbers (bf16 cache, whose values fix the operands' type): one alone would make the output's error 1.4 times
// that of its own rounding, the second costs 1 % of the time.  e4m3 codes are widened exactly to fp16; every query head is scaled by a power of two into fp16's range first.
#include "internal.h"

namespace dsuf {

constexpr int KID_DECODE = 8;
constexpr int AD_WARPS = 4;
constexpr int AD_THREADS = AD_WARPS * 32;
constexpr int AD_STAGES = 3;
constexpr int AD_HALF = 4096;                              // bytes of keys (and of values) in a warp's stage
constexpr int AD_RING = AD_WARPS * AD_STAGES * 2 * AD_HALF;
constexpr int AD_PART = 16 * 128;                          // floats of one partial output
constexpr int AD_JOIN = 16;                                // partials whose loads are in flight together when a piece is joined
constexpr int AD_SEGMENT_SHIFT = 2;                        // log2 of the units of a segment when there are few
constexpr unsigned AD_SOLO_UNITS = 4;                      // a warp per piece: pieces of at most so many units, and one for every CTA that the GPU holds
constexpr float AD_UNSET = -3.4028234663852886e38f;         // no finite score is below it
constexpr float AD_TRIGGER = 15.f, AD_HEADROOM = 7.f;

struct DecodeArgs {
    const bf16* q;
    bf16* out;
    float* lse;
    int ldq, ldo, b, q_heads, kv_heads, group, blocks;     // blocks: blocks of 8 NT heads in a group
    const int *table, *lens;
    int max_pages, n_pages, page_shift, window;
    const uint8_t *ck, *cv;
    const float *k_scale, *v_scale;
    long long page_bytes;
    float scale_log2;
    float *part, *part_ml;                                 // [CTA][2][16][128] and [CTA][2][16][2]
    int* counter;                                          // [CTA]
    unsigned solo_from;                                    // pieces
    DevStatus* status;
};

DSUF_DEV void cp_async16_zfill(uint32_t dst, const void* src, bool take) {
    const int n = take ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
DSUF_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
DSUF_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
DSUF_DEV void ldsm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
DSUF_DEV void ldsm4t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
DSUF_DEV uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool HALF>
DSUF_DEV void mma_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DSUF_DEV uint32_t e4m3x2_to_f16x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
DSUF_DEV float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool HALF>
DSUF_DEV uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int D, bool FP8, int NT>
struct DecodeShape {
    static constexpr int ROW = D * (FP8 ? 1 : 2);          // bytes of a token's key
    static constexpr int CH = AD_HALF / ROW;               // tokens of a warp's stage
    static constexpr int SUBS = CH / 16;
    static constexpr int CH_SHIFT = CH == 16 ? 4 : CH == 32 ? 5 : 6;
    static constexpr int UNIT = AD_WARPS * CH;
    static_assert(CH == 1 << CH_SHIFT && AD_WARPS == 4, "units are powers of two");
    static constexpr int PIECES = ROW / 16;                // 16-byte columns of a row
    static constexpr int ROWS = 8 * NT;                    // query heads of a block
    static constexpr int SMEM = AD_RING + AD_WARPS * 8 * D * 4;
};

// Byte offset of 16-byte column c of row r: the columns of a 128-byte line are permuted by the line's index, so that eight
// consecutive rows' same column fall into eight different bank groups.
template <int ROW>
DSUF_DEV uint32_t ring_at(int r, int c) {
    if constexpr (ROW == 256) return r * 256 + ((c ^ (r & 7)) << 4);
    else if constexpr (ROW == 128) return r * 128 + ((c ^ (r & 7)) << 4);
    else return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ ((r >> 1) & 7)) << 4);
}

// A place in the sequence of all units: sequence, (kv head, head block), unit inside the piece; the sequence's visible range.
struct UnitAt {
    int seq, hb, u, nu, beg, len;
};

// (units of 2^unit tokens)
DSUF_DEV void visible_range(const DecodeArgs& a, int seq, int unit, int& beg, int& len, int& nu) {
    len = seq < a.b ? __ldg(a.lens + seq) : 0;
    const int cap = a.max_pages << a.page_shift;
    len = min(max(len, 0), cap);
    beg = a.window > 0 ? max(0, len - a.window) : 0;
    nu = len > 0 ? (len - (beg & ~15) + (1 << unit) - 1) >> unit : 0;
}
DSUF_DEV void next_unit(const DecodeArgs& a, UnitAt& p, int unit) {
    if (++p.u < p.nu) return;
    p.u = 0;
    if (++p.hb < a.kv_heads * a.blocks) return;
    p.hb = 0;
    do {
        ++p.seq;
        visible_range(a, p.seq, unit, p.beg, p.len, p.nu);
    } while (p.seq < a.b && p.nu == 0);
}

// Rows of sequences that see nothing.
template <int D>
DSUF_DEV void empty_rows(const DecodeArgs& a) {
    for (int i = blockIdx.x; i < a.b; i += gridDim.x) {
        const int len = __ldg(a.lens + i);
        if (len > (a.max_pages << a.page_shift) && threadIdx.x == 0) report(a.status, DEVERR_BAD_PLAN, KID_DECODE, 1);
        if (len > 0) continue;
        for (int j = threadIdx.x; j < a.q_heads * D / 8; j += AD_THREADS)
            *reinterpret_cast<uint4*>(a.out + (size_t)i * a.ldo + (size_t)j * 8) = make_uint4(0, 0, 0, 0);
        if (a.lse)
            for (int j = threadIdx.x; j < a.q_heads; j += AD_THREADS) a.lse[(size_t)i * a.q_heads + j] = -INFINITY;
    }
}

// The sum of a cut piece's partials, in CTA order.  A warp takes two rows (query heads) at a time and the partials 32 at a time: each lane reads one
// partial's reference point and sum and turns it into a weight, while the first AD_JOIN outputs of each row are on their way.  (A chain that moves the
// reference from partial to partial took 17800 cycles for 37 partials; a load of what another SM has written takes about 1000.)
template <int D>
DSUF_DEV void join_piece(const DecodeArgs& a, int first, int last, int heads, int seq, int head0, float out_scale) {
    constexpr int V = D / 32;                              // columns of a lane
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = last - first + 1;
    auto slot = [&](int f) { return (size_t)(first + f) * 2 + (f == 0 ? 1 : 0); };
    for (int r0 = warp * 2; r0 < heads; r0 += AD_WARPS * 2) {
        const int rows[2] = {r0, min(r0 + 1, heads - 1)};  // (an odd last row is done twice)
        float top[2] = {AD_UNSET, AD_UNSET}, l[2] = {0.f, 0.f}, acc[2][V];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[0][e] = acc[1][e] = 0.f;
        for (int f0 = 0; f0 < n; f0 += 32) {
            const int here = min(32, n - f0);
            float2 ml[2];
            float w[2], v[2][AD_JOIN][V];
#pragma unroll
            for (int q = 0; q < 2; ++q) ml[q] = lane < here ? __ldcg(reinterpret_cast<const float2*>(a.part_ml + slot(f0 + lane) * 32 + 2 * rows[q])) : make_float2(0.f, 0.f);
            for (int f = 0; f < here; f += AD_JOIN) {
#pragma unroll
                for (int j = 0; j < AD_JOIN; ++j) {
                    const float* p = a.part + slot(f0 + f + j) * AD_PART + lane * V;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        if (f + j >= here) {
#pragma unroll
                            for (int e = 0; e < V; ++e) v[q][j][e] = 0.f;
                        } else if constexpr (V == 4) {
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(p + rows[q] * D));
                            v[q][j][0] = x.x; v[q][j][1] = x.y; v[q][j][2] = x.z; v[q][j][3] = x.w;
                        } else {
                            const float2 x = __ldcg(reinterpret_cast<const float2*>(p + rows[q] * D));
                            v[q][j][0] = x.x; v[q][j][1] = x.y;
                        }
                    }
                }
                if (f == 0) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float to = ml[q].y != 0.f ? fmaxf(top[q], ml[q].x) : top[q];
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
                        const float by = exp2_approx(top[q] - to);
                        top[q] = to;
                        w[q] = ml[q].y != 0.f ? exp2_approx(ml[q].x - to) : 0.f;
                        l[q] = l[q] * by + w[q] * ml[q].y;
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[q][e] *= by;
                    }
                }
#pragma unroll
                for (int j = 0; j < AD_JOIN; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float wf = __shfl_sync(0xffffffffu, w[q], f + j);     // (0 beyond the last one)
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[q][e] += wf * v[q][j][e];
                    }
            }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l[q] += __shfl_xor_sync(0xffffffffu, l[q], o);
            const float inv = l[q] == 0.f ? 0.f : out_scale / l[q];
            bf16* dst = a.out + (size_t)seq * a.ldo + (size_t)(head0 + rows[q]) * D + lane * V;
            if constexpr (V == 4)
                *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<false>(acc[q][0] * inv, acc[q][1] * inv), pack2<false>(acc[q][2] * inv, acc[q][3] * inv));
            else
                *reinterpret_cast<uint32_t*>(dst) = pack2<false>(acc[q][0] * inv, acc[q][1] * inv);
            if (a.lse && lane == 0)
                a.lse[(size_t)seq * a.q_heads + head0 + rows[q]] = l[q] == 0.f ? -INFINITY : (top[q] + log2f(l[q])) * 0.6931471805599453f;
        }
    }
}

template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(AD_THREADS, 2) attn_decode_kernel(const DecodeArgs a) {
    using S = DecodeShape<D, FP8, NT>;
    constexpr int KS = D / 16;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* merge = reinterpret_cast<float*>(smem + AD_RING);       // [warp][8][D]
    __shared__ float s_ref[AD_WARPS][8], s_sum[AD_WARPS][8];
    __shared__ int s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int quad = lane & 3, row8 = lane >> 2;
    pdl_wait();
    pdl_launch_dependents();

    // What is dealt are segments of 2^seg units: of one unit; of 2^AD_SEGMENT_SHIFT where the GPU would get fewer than that many units per CTA (then a
    // piece's parts begin with the CTAs, few have to be joined, and a short piece stays whole); of whole pieces, and to warps instead of CTAs
    // (`solo`: a unit is then the CH tokens of one warp), where all pieces are short and many.  Every warp finds its range by itself: the lanes sum
    // up a share of the sequences each.  (All numbers of units are below 2^31: the host has seen to that.)
    const int HB = a.kv_heads * a.blocks;
    const int share = (a.b + 31) / 32, i0 = min(a.b, lane * share), i1 = min(a.b, i0 + share);
    unsigned mine, longest;
    auto sum_up = [&](int unit, int seg) {
        mine = longest = 0;
        for (int i = i0; i < i1; ++i) {
            int beg, len, nu;
            visible_range(a, i, unit, beg, len, nu);
            mine += (unsigned)(((nu + (1 << seg) - 1) >> seg) * HB);
            longest = max(longest, (unsigned)nu);
        }
        unsigned upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        return upto;
    };
    int unit = S::CH_SHIFT + 2, seg = 0;
    unsigned upto = sum_up(unit, 0);
    const bool few = __shfl_sync(0xffffffffu, upto, 31) < gridDim.x << AD_SEGMENT_SHIFT;
    bool solo = (unsigned)(a.b * HB) >= a.solo_from && __reduce_max_sync(0xffffffffu, longest) <= AD_SOLO_UNITS;
    if (solo) {
        const unsigned pieces = sum_up(unit, 20);
        solo = __shfl_sync(0xffffffffu, pieces, 31) >= a.solo_from;
        upto = pieces;
    }
    if (solo) {
        unit = S::CH_SHIFT;
        seg = 20;
    } else if (few) {
        seg = AD_SEGMENT_SHIFT;
        upto = sum_up(unit, seg);
    } else {
        upto = sum_up(unit, 0);
    }
    const int own = solo ? 0 : warp * S::CH;            // the warp's tokens inside a unit
    const unsigned total = __shfl_sync(0xffffffffu, upto, 31);
    const unsigned worker = solo ? warp * gridDim.x + blockIdx.x : blockIdx.x, workers = solo ? gridDim.x * AD_WARPS : gridDim.x;
    const unsigned used = min(workers, total);          // CTAs, or warps, that get work
    if (worker >= used) {
        empty_rows<D>(a);
        return;
    }
    // the first `more` CTAs take base + 1 segments, the others base
    const unsigned base = total / used, more = total % used;
    const unsigned s0 = base * worker + min(worker, more), s1 = s0 + base + (worker < more ? 1 : 0);
    auto cta_of = [&](unsigned segment) {
        const unsigned cut = more * (base + 1);
        return segment < cut ? segment / (base + 1) : more + (segment - cut) / base;
    };
    UnitAt at;
    {
        const unsigned past = __ballot_sync(0xffffffffu, upto > s0);
        const int owner = __ffs(past) - 1;
        if (lane == owner) {
            unsigned left = s0 - (upto - mine);
            at.seq = i0;
            unsigned n;
            for (;;) {
                visible_range(a, at.seq, unit, at.beg, at.len, at.nu);
                n = (unsigned)((at.nu + (1 << seg) - 1) >> seg);
                if (left < n * HB) break;
                left -= n * HB;
                ++at.seq;
            }
            at.hb = (int)(left / n);
            at.u = (int)(left % n) << seg;
        }
        at.seq = __shfl_sync(0xffffffffu, at.seq, owner);
        at.hb = __shfl_sync(0xffffffffu, at.hb, owner);
        at.u = __shfl_sync(0xffffffffu, at.u, owner);
        at.nu = __shfl_sync(0xffffffffu, at.nu, owner);
        at.beg = __shfl_sync(0xffffffffu, at.beg, owner);
        at.len = __shfl_sync(0xffffffffu, at.len, owner);
    }

    const uint32_t ring = smem_u32(smem) + warp * AD_STAGES * 2 * AD_HALF;
    // this lane's destinations inside a half stage: 8 vectors, 512 bytes of source apart
    uint32_t dst_at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dst_at[i] = ring_at<S::ROW>((i * 32 + lane) / S::PIECES, (i * 32 + lane) % S::PIECES);

    struct Pages { int id[S::SUBS]; };
    auto look_up = [&](const UnitAt& p) {
        Pages r;
        const int t0 = (p.beg & ~15) + (p.u << unit) + own;
#pragma unroll
        for (int s = 0; s < S::SUBS; ++s)
            r.id[s] = t0 + 16 * s < p.len ? __ldg(a.table + (size_t)p.seq * a.max_pages + ((t0 + 16 * s) >> a.page_shift)) : 0;
        return r;
    };
    auto issue = [&](const UnitAt& p, int stage, const Pages& pages) {
        const int t0 = (p.beg & ~15) + (p.u << unit) + own;
        const int kvh = p.hb / a.blocks;
        const uint32_t kdst = ring + stage * 2 * AD_HALF, vdst = kdst + AD_HALF;
#pragma unroll
        for (int s = 0; s < S::SUBS; ++s) {
            const int ts = t0 + 16 * s;
            const bool some = ts < p.len;    // (ts + 16 > beg for every unit)
            int page = pages.id[s];
            const bool good = page >= 0 && page < a.n_pages;
            if (!good) {
                if (lane == 0) report(a.status, DEVERR_BAD_PLAN, KID_DECODE, 2);
                page = 0;
            }
            const size_t off = (size_t)page * a.page_bytes +
                               (((size_t)kvh << a.page_shift) + (size_t)(ts & ((1 << a.page_shift) - 1))) * S::ROW + lane * 16;
            constexpr int PER = 8 / S::SUBS;   // vectors of a lane inside 16 tokens
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = s * PER + j;
                const int t = t0 + (i * 32 + lane) / S::PIECES;
                const bool take = some && good && t >= p.beg && t < p.len;
                cp_async16_zfill(kdst + dst_at[i], a.ck + off + j * 512, take);
                cp_async16_zfill(vdst + dst_at[i], a.cv + off + j * 512, take);
            }
        }
    };

    // The loads walk ahead of the products; both count the segments that the CTA has left, and a step says whether it ended one.
    UnitAt ahead = at;
    unsigned to_load = s1 - s0, to_do = to_load;
    auto step = [&](UnitAt& p) {
        const bool ends = p.u + 1 == p.nu || ((p.u + 1) & ((1 << seg) - 1)) == 0;
        next_unit(a, p, unit);
        return ends ? 1u : 0u;
    };
    int fill = 0, use = 0;
    {
        // (the first units' pages are looked up together: the chain lengths -> pages -> keys is what a short call waits for)
        UnitAt first[AD_STAGES - 1];
        Pages pages[AD_STAGES - 1];
        bool some[AD_STAGES - 1];
#pragma unroll
        for (int i = 0; i < AD_STAGES - 1; ++i) {
            first[i] = ahead;
            some[i] = to_load > 0;
            if (some[i]) {
                pages[i] = look_up(ahead);
                to_load -= step(ahead);
            }
        }
#pragma unroll
        for (int i = 0; i < AD_STAGES - 1; ++i) {
            if (some[i]) issue(first[i], fill, pages[i]);
            cp_async_commit();
            if (++fill == AD_STAGES) fill = 0;
        }
    }

    while (to_do > 0) {
        // ---------------- one piece, or this CTA's part of it ----------------
        const int kvh = at.hb / a.blocks, hblk = at.hb % a.blocks;
        const int head0 = kvh * a.group + hblk * S::ROWS;              // first query head of the block
        const int heads = min(S::ROWS, a.group - hblk * S::ROWS);
        const unsigned seg_at = (unsigned)(at.u >> seg), seg_all = (unsigned)((at.nu + (1 << seg) - 1) >> seg);     // in the piece
        const unsigned segs = min(to_do, seg_all - seg_at);
        const int frag = min((int)(segs << seg), at.nu - at.u);         // units
        // query operand: column n = head, k = 16 columns of the head per step
        uint32_t qf[KS][NT][2];
        float sl2[NT][2];        // log2(e) times the scale of the scores, of the heads 2 quad and 2 quad + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int h = nt * 8 + row8;
            const bf16* src = a.q + (size_t)at.seq * a.ldq + (size_t)(head0 + h) * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                // bf16: columns 2 quad and 2 quad + 8 of the step; e4m3: 4 quad .. 4 quad + 3, as the widened keys lie
                const int c0 = ks * 16 + (FP8 ? 4 * quad : 2 * quad);
                const int c1 = ks * 16 + (FP8 ? 4 * quad + 2 : 2 * quad + 8);
                qf[ks][nt][0] = h < heads ? *reinterpret_cast<const uint32_t*>(src + c0) : 0u;
                qf[ks][nt][1] = h < heads ? *reinterpret_cast<const uint32_t*>(src + c1) : 0u;
            }
        }
        if constexpr (FP8) {
            // a head's largest finite magnitude -> a power of two that brings it to about 2^14
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                uint32_t top = 0;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t m = (qf[ks][nt][j] >> (16 * e)) & 0x7fffu;
                            if (m < 0x7f80u) top = max(top, m);
                        }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int shift = min(max(14 - ((int)(top >> 7) - 127), -120), 120);
                const float up = __uint_as_float((uint32_t)(shift + 127) << 23);
                const float scale = a.scale_log2 * __uint_as_float((uint32_t)(127 - shift) << 23) * (a.k_scale ? __ldg(a.k_scale + kvh) : 1.f);
                sl2[nt][0] = __shfl_sync(0xffffffffu, scale, quad * 8);
                sl2[nt][1] = __shfl_sync(0xffffffffu, scale, quad * 8 + 4);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        qf[ks][nt][j] = pack2<true>(__uint_as_float(qf[ks][nt][j] << 16) * up, __uint_as_float(qf[ks][nt][j] & 0xffff0000u) * up);
            }
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sl2[nt][0] = sl2[nt][1] = a.scale_log2;
        }
        float o[KS][NT][4], ref[NT][2], sum[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            ref[nt][0] = ref[nt][1] = AD_UNSET;
            sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[ks][nt][e] = 0.f;
        }
        int t0 = (at.beg & ~15) + (at.u << unit) + own;
        for (int f = 0; f < frag; ++f, t0 += 1 << unit) {
            cp_async_wait<AD_STAGES - 2>();
            __syncwarp();   // the stage is full, and every lane is through with the stage that is filled next
            if (to_load > 0) {
                issue(ahead, fill, look_up(ahead));
                to_load -= step(ahead);
            }
            cp_async_commit();
            if (++fill == AD_STAGES) fill = 0;
            const uint32_t kst = ring + use * 2 * AD_HALF, vst = kst + AD_HALF;
            if (++use == AD_STAGES) use = 0;
            if (t0 >= at.len) continue;
            const bool edge = t0 < at.beg || t0 + S::CH > at.len;
#pragma unroll
            for (int s = 0; s < S::SUBS; ++s) {
                if (edge && t0 + 16 * s >= at.len) break;
                float st[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st[nt][e] = 0.f;
                // S^T (16 tokens x heads): rows 0-7 / 8-15 and two 16-byte columns per ldmatrix
                const int kr = s * 16 + (lane & 15);
                if constexpr (!FP8) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t kf[4];
                        ldsm4(kf, kst + ring_at<S::ROW>(kr, ks * 2 + (lane >> 4)));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816<false>(st[nt], kf, qf[ks][nt][0], qf[ks][nt][1]);
                    }
                } else {
#pragma unroll
                    for (int kk = 0; kk < KS / 2; ++kk) {
                        uint32_t raw[4];
                        ldsm4(raw, kst + ring_at<S::ROW>(kr, kk * 2 + (lane >> 4)));
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t kf[4] = {e4m3x2_to_f16x2((uint16_t)raw[2 * e]), e4m3x2_to_f16x2((uint16_t)raw[2 * e + 1]),
                                                    e4m3x2_to_f16x2((uint16_t)(raw[2 * e] >> 16)), e4m3x2_to_f16x2((uint16_t)(raw[2 * e + 1] >> 16))};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_16816<true>(st[nt], kf, qf[2 * kk + e][nt][0], qf[2 * kk + e][nt][1]);
                        }
                    }
                }
                if (edge) {
                    const int ta = t0 + 16 * s + row8, tb = ta + 8;
                    const bool va = ta >= at.beg && ta < at.len, vb = tb >= at.beg && tb < at.len;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        st[nt][0] = va ? st[nt][0] * sl2[nt][0] : -INFINITY;
                        st[nt][1] = va ? st[nt][1] * sl2[nt][1] : -INFINITY;
                        st[nt][2] = vb ? st[nt][2] * sl2[nt][0] : -INFINITY;
                        st[nt][3] = vb ? st[nt][3] * sl2[nt][1] : -INFINITY;
                    }
                } else {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) st[nt][e] *= sl2[nt][e & 1];
                }
                bool over = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    over |= fmaxf(st[nt][0], st[nt][2]) > ref[nt][0] + AD_TRIGGER;
                    over |= fmaxf(st[nt][1], st[nt][3]) > ref[nt][1] + AD_TRIGGER;
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(st[nt][e], st[nt][e + 2]);
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                            if (top > ref[nt][e] + AD_TRIGGER) {
                                const float to = top - AD_HEADROOM;
                                const float by = exp2_approx(ref[nt][e] - to);
                                ref[nt][e] = to;
                                sum[nt][e] *= by;
#pragma unroll
                                for (int ks = 0; ks < KS; ++ks) {
                                    o[ks][nt][e] *= by;
                                    o[ks][nt][e + 2] *= by;
                                }
                            }
                        }
                }
                // bf16: p as its leading bits and the rest, which gets 2^-23 p on top so that both parts are positive where p is: a visible infinity times
                // them is infinite (0 x infinity, or infinity - infinity, would be NaN)
                uint32_t pf[NT][2], pr[NT][2];
                auto front = [](float x, float y) { return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632); };
                auto rest = [](float x) { return fmaf(x, 1.f + 0x1p-23f, -__uint_as_float(__float_as_uint(x) & 0xffff0000u)); };
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = exp2_approx(st[nt][e] - ref[nt][e & 1]);
                    sum[nt][0] += p[0] + p[2];
                    sum[nt][1] += p[1] + p[3];
                    if constexpr (FP8) {
                        pf[nt][0] = transpose8x8(pack2<true>(p[0], p[1]));
                        pf[nt][1] = transpose8x8(pack2<true>(p[2], p[3]));
                    } else {
                        pf[nt][0] = transpose8x8(front(p[0], p[1]));
                        pf[nt][1] = transpose8x8(front(p[2], p[3]));
                        pr[nt][0] = transpose8x8(pack2<false>(rest(p[0]), rest(p[1])));
                        pr[nt][1] = transpose8x8(pack2<false>(rest(p[2]), rest(p[3])));
                    }
                }
                // O^T (D x heads) += V^T (D x 16 tokens) P^T
                if constexpr (!FP8) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t vf[4];
                        ldsm4t(vf, vst + ring_at<S::ROW>(s * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_16816<false>(o[ks][nt], vf, pf[nt][0], pf[nt][1]);
                            mma_16816<false>(o[ks][nt], vf, pr[nt][0], pr[nt][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int kk = 0; kk < KS / 2; ++kk) {
                        uint32_t raw[4];   // tokens 0-7 / 8-15 of 16 columns, then of the next 16; a word holds columns (2i, 2i + 1) of two tokens
                        ldsm4t(raw, vst + ring_at<S::ROW>(kr, kk * 2 + (lane >> 4)));
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t lo = __byte_perm(raw[2 * e], 0, 0x3120), hi = __byte_perm(raw[2 * e + 1], 0, 0x3120);
                            const uint32_t vf[4] = {e4m3x2_to_f16x2((uint16_t)lo), e4m3x2_to_f16x2((uint16_t)(lo >> 16)), e4m3x2_to_f16x2((uint16_t)hi),
                                                    e4m3x2_to_f16x2((uint16_t)(hi >> 16))};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_16816<true>(o[2 * kk + e][nt], vf, pf[nt][0], pf[nt][1]);
                        }
                    }
                }
            }
        }

        const float out_scale = FP8 && a.v_scale ? __ldg(a.v_scale + kvh) : 1.f;
        if (solo) {
            // ---------------- the warp's own piece ----------------
            float* mw = merge + warp * 8 * D;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (nt * 8 >= heads) break;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float l = sum[nt][e];
                    l += __shfl_xor_sync(0xffffffffu, l, 4);
                    l += __shfl_xor_sync(0xffffffffu, l, 8);
                    l += __shfl_xor_sync(0xffffffffu, l, 16);
                    const float inv = l == 0.f ? 0.f : out_scale / l;
                    const int h = nt * 8 + 2 * quad + e;
                    if (a.lse && row8 == 0 && h < heads) a.lse[(size_t)at.seq * a.q_heads + head0 + h] = l == 0.f ? -INFINITY : (ref[nt][e] + log2f(l)) * 0.6931471805599453f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int col = FP8 ? ks * 16 + 2 * row8 + half : ks * 16 + row8 + 8 * half;
                            mw[(2 * quad + e) * D + col] = o[ks][nt][e + 2 * half] * inv;
                        }
                }
                __syncwarp();
#pragma unroll
                for (int i = lane; i < 8 * D / 4; i += 32) {
                    const int r = i / (D / 4), c = (i % (D / 4)) * 4;
                    const float4 v = *reinterpret_cast<const float4*>(mw + r * D + c);
                    if (nt * 8 + r < heads)
                        *reinterpret_cast<uint2*>(a.out + (size_t)at.seq * a.ldo + (size_t)(head0 + nt * 8 + r) * D + c) =
                            make_uint2(pack2<false>(v.x, v.y), pack2<false>(v.z, v.w));
                }
                __syncwarp();
            }
            to_do -= segs;
            at.u += frag - 1;
            next_unit(a, at, unit);
            continue;
        }
        // ---------------- the four warps' parts of the piece ----------------
        const bool whole = frag == at.nu;
        const bool leads = at.u + frag < at.nu && at.u == 0;     // first CTA of a cut piece: its second slot
        const unsigned piece0 = s1 - to_do - seg_at;             // the piece's first segment
        float* part = a.part + ((size_t)blockIdx.x * 2 + (leads ? 1 : 0)) * AD_PART;
        float* part_ml = a.part_ml + ((size_t)blockIdx.x * 2 + (leads ? 1 : 0)) * 32;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt * 8 >= heads) break;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = sum[nt][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (row8 == 0) {
                    s_ref[warp][2 * quad + e] = ref[nt][e];
                    s_sum[warp][2 * quad + e] = l;
                }
            }
            float* mw = merge + warp * 8 * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int col = FP8 ? ks * 16 + 2 * row8 + (e >> 1) : ks * 16 + row8 + 8 * (e >> 1);
                    mw[(2 * quad + (e & 1)) * D + col] = o[ks][nt][e];
                }
            __syncthreads();
            for (int i = tid; i < 8 * D / 4; i += AD_THREADS) {
                const int r = i / (D / 4), c = (i % (D / 4)) * 4;
                float top = s_ref[0][r];
#pragma unroll
                for (int w = 1; w < AD_WARPS; ++w) top = fmaxf(top, s_ref[w][r]);
                float l = 0.f;
                float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
                for (int w = 0; w < AD_WARPS; ++w) {
                    const float f = s_sum[w][r] == 0.f ? 0.f : exp2_approx(s_ref[w][r] - top);
                    const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + r) * D + c);
                    l += f * s_sum[w][r];
                    acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
                }
                const int h = nt * 8 + r;
                if (h < heads) {
                    if (whole) {
                        const float inv = l == 0.f ? 0.f : out_scale / l;
                        *reinterpret_cast<uint2*>(a.out + (size_t)at.seq * a.ldo + (size_t)(head0 + h) * D + c) =
                            make_uint2(pack2<false>(acc.x * inv, acc.y * inv), pack2<false>(acc.z * inv, acc.w * inv));
                        if (a.lse && c == 0) a.lse[(size_t)at.seq * a.q_heads + head0 + h] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
                    } else {
                        __stcg(reinterpret_cast<float4*>(part + h * D + c), acc);
                        if (c == 0) __stcg(reinterpret_cast<float2*>(part_ml + 2 * h), make_float2(top, l));
                    }
                }
            }
            __syncthreads();
        }
        if (!whole) {
            // the CTAs that hold units of this piece: first .. last; the counter of the first one counts them
            const int first = (int)cta_of(piece0), last = (int)cta_of(piece0 + seg_all - 1);
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                s_last = atomicAdd(a.counter + first, 1) == last - first;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                join_piece<D>(a, first, last, heads, at.seq, head0, out_scale);
                if (tid == 0) a.counter[first] = 0;
            }
        }
        to_do -= segs;
        at.u += frag - 1;
        next_unit(a, at, unit);
    }
    cp_async_wait<0>();
    empty_rows<D>(a);
}

template <int D, bool FP8, int NT>
static int decode_attr(dsuf_ctx* ctx) {
    cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<D, FP8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeShape<D, FP8, NT>::SMEM);
    return e == cudaSuccess ? DSUF_OK : cuda_fail(ctx, e, "cudaFuncSetAttribute(attn_decode)");
}
int attn_decode_setup(dsuf_ctx* ctx) {
    int rc = 0;
    if (!rc) rc = decode_attr<64, false, 1>(ctx);
    if (!rc) rc = decode_attr<64, false, 2>(ctx);
    if (!rc) rc = decode_attr<64, true, 1>(ctx);
    if (!rc) rc = decode_attr<64, true, 2>(ctx);
    if (!rc) rc = decode_attr<128, false, 1>(ctx);
    if (!rc) rc = decode_attr<128, false, 2>(ctx);
    if (!rc) rc = decode_attr<128, true, 1>(ctx);
    if (!rc) rc = decode_attr<128, true, 2>(ctx);
    return rc;
}

static int decode_ctas(dsuf_ctx* ctx) { return 2 * ctx->sm_count; }

template <int D, bool FP8, int NT>
static int decode_launch(dsuf_ctx* ctx, cudaStream_t stream, DecodeArgs& a) {
    using S = DecodeShape<D, FP8, NT>;
    a.blocks = (a.group + S::ROWS - 1) / S::ROWS;
    // no more CTAs than units that the block table could hold (their number is only known on the device)
    const long long cap = (long long)a.b * a.kv_heads * a.blocks * ((((long long)a.max_pages << a.page_shift) + 15 + S::UNIT - 1) / S::UNIT);
    DSUF_REQUIRE(ctx, cap < (1ll << 31), "attn_decode: b * kv_heads * positions of the block table is too large (%lld units of work)", cap);
    DSUF_REQUIRE_DEVICE(ctx, "attn_decode");
    const int grid = (int)(cap < decode_ctas(ctx) ? cap : decode_ctas(ctx));
    return launch(ctx, stream, attn_decode_kernel<D, FP8, NT>, dim3(grid), dim3(AD_THREADS), (size_t)S::SMEM, a);
}

}  // namespace dsuf

using namespace dsuf;

extern "C" {

size_t dsuf_attn_workspace_bytes(dsuf_ctx* ctx) {
    if (!ctx) return 0;
    return (size_t)decode_ctas(ctx) * (2 * (AD_PART + 32) * sizeof(float) + 16);
}

int32_t dsuf_attn_workspace_init(dsuf_ctx* ctx, void* stream, uint64_t workspace, size_t bytes) {
    if (!ctx) return DSUF_E_BADARG;
    DSUF_REQUIRE(ctx, workspace && (workspace & 15) == 0 && bytes >= dsuf_attn_workspace_bytes(ctx), "attn_workspace_init: need %zu bytes, 16-byte aligned",
                 dsuf_attn_workspace_bytes(ctx));
    DSUF_REQUIRE_DEVICE(ctx, "attn_workspace_init");
    cudaError_t e = cudaMemsetAsync((void*)workspace, 0, dsuf_attn_workspace_bytes(ctx), (cudaStream_t)stream);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaMemsetAsync(attention workspace)");
    return DSUF_OK;
}

int32_t dsuf_attn_decode(dsuf_ctx* ctx, void* stream, const dsuf_kv_cache* cache, uint64_t q, int32_t ldq, int32_t q_heads, int32_t b,
                         uint64_t block_table, int32_t max_pages, uint64_t seq_lens, float scale, int32_t window, uint64_t out,
                         int32_t ldo, uint64_t lse, uint64_t workspace) {
    if (!ctx) return DSUF_E_BADARG;
    int rc = check_kv_cache(ctx, "attn_decode", cache);
    if (rc) return rc;
    const int D = cache->head_dim;
    DSUF_REQUIRE(ctx, b >= 0 && max_pages >= 1 && (long long)max_pages * cache->page_size <= 0x7fff0000ll,
                 "attn_decode: b >= 0, max_pages >= 1 and at most 2^31 - 65536 positions");
    DSUF_REQUIRE(ctx, q_heads >= 1 && q_heads <= 4096 && q_heads % cache->kv_heads == 0, "attn_decode: q_heads (%d) must be a multiple of kv_heads (%d), at most 4096",
                 q_heads, cache->kv_heads);
    DSUF_REQUIRE(ctx, ldq >= q_heads * D && ldq % 8 == 0 && ldo >= q_heads * D && ldo % 8 == 0,
                 "attn_decode: ldq and ldo must be multiples of 8 and hold q_heads * head_dim elements");
    DSUF_REQUIRE(ctx, window >= 0 && scale > 0.f && scale - scale == 0.f, "attn_decode: window must be >= 0, scale positive and finite");
    if (b == 0) return DSUF_OK;
    DSUF_REQUIRE(ctx, q && out && block_table && seq_lens && workspace && (q & 15) == 0 && (out & 15) == 0 && (block_table & 3) == 0 &&
                 (seq_lens & 3) == 0 && (lse & 3) == 0 && (workspace & 15) == 0, "attn_decode: null or misaligned pointer (q, out, workspace 16 bytes, indexes and lse 4)");
    const long long width = (long long)q_heads * D, lse_bytes = 4ll * b * q_heads;
    DSUF_REQUIRE(ctx, rows_in_place(out, ldo, q, ldq, b) || !rows_overlap(out, ldo, width, q, ldq, width, b), "attn_decode: out must be q itself, row for row, or share no memory with it");
    DSUF_REQUIRE(ctx, !lse || (!block_meets_rows(lse, lse_bytes, q, ldq, width, b) && !block_meets_rows(lse, lse_bytes, out, ldo, width, b)),
                 "attn_decode: lse must share no memory with q and out");
    DecodeArgs a;
    memset(&a, 0, sizeof(a));
    a.q = (const bf16*)q; a.out = (bf16*)out; a.lse = (float*)lse;
    a.ldq = ldq; a.ldo = ldo; a.b = b; a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.group = q_heads / cache->kv_heads;
    a.table = (const int*)block_table; a.lens = (const int*)seq_lens;
    a.max_pages = max_pages; a.n_pages = cache->n_pages; a.page_shift = __builtin_ctz((unsigned)cache->page_size); a.window = window;
    a.ck = (const uint8_t*)cache->k; a.cv = (const uint8_t*)cache->v;
    a.k_scale = (const float*)cache->k_scale; a.v_scale = (const float*)cache->v_scale;
    const bool fp8 = cache->dtype == DSUF_KV_E4M3;
    a.page_bytes = cache->page_stride * (fp8 ? 1 : 2);
    a.scale_log2 = scale * 1.4426950408889634f;
    const int n = decode_ctas(ctx);
    a.part = (float*)workspace;
    a.part_ml = a.part + (size_t)n * 2 * AD_PART;
    a.counter = (int*)(a.part_ml + (size_t)n * 2 * 32);
    a.solo_from = (unsigned)n;
    a.status = ctx->dev_status;
    cudaStream_t s = (cudaStream_t)stream;
    if (a.group <= 8) {   // one column block of 8 heads holds the group; larger groups go by 16 (half the passes over the cache)
        if (D == 64) return fp8 ? decode_launch<64, true, 1>(ctx, s, a) : decode_launch<64, false, 1>(ctx, s, a);
        return fp8 ? decode_launch<128, true, 1>(ctx, s, a) : decode_launch<128, false, 1>(ctx, s, a);
    }
    if (D == 64) return fp8 ? decode_launch<64, true, 2>(ctx, s, a) : decode_launch<64, false, 2>(ctx, s, a);
    return fp8 ? decode_launch<128, true, 2>(ctx, s, a) : decode_launch<128, false, 2>(ctx, s, a);
}

}  // extern "C"
