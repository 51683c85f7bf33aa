// sx8_kv4.hip -- the paged 4-bit KV cache: writer, reader and attention (include/sx8_paged.h).
#include "sx8_kv4_core.h"

namespace sx8 {
namespace {

// ---- append ------------------------------------------------------------------------------------
// A work-group encodes the new rows of one block of one head, so that no word of the cache has two writers.
// Eight lanes hold a group of 64 values (16 bytes each): minimum and maximum by three lane exchanges, then each
// lane's eight levels.  K's eight levels of a lane are one word; V's word holds eight tokens of a dimension, so V's
// levels meet in LDS, and a word with tokens of earlier calls keeps their bits.
// 13081 rows of 8 heads of 128 take 20 us (69 MB, 3.5 TB/s; the VALU is busy 56% of the time, 1.7 rounds of work-groups), a
// row of each of 64 slots 4.8, where the chain of lengths, table and rows is all there is.

template <int HD, bool kBf16>
__global__ __launch_bounds__(256) void k_kv4_append(const Kv4Pool p, const RowsIn in) {
    constexpr int kBB = kv4_block_bytes(HD), CPR = HD / 8, NI = 32 * CPR / 256;   // chunks of a row; rounds of K or V
    __shared__ __align__(8) uint8_t lv[32][HD + 8];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    Touched t;
    if (!find_touched(p, blockIdx.x, pre, &t)) return;
    const int head = blockIdx.y, tid = threadIdx.x;
    const int64_t off = block_offset(p, t.slot, head, t.block, kBB);
    const int nt = t.t1 - t.t0;
    // every row of the block's share is requested before the first is encoded (and while the page number is on its way)
    constexpr int kStep = 256 / CPR;                                // rows between a thread's chunks
    u32x4 raw[2][NI];
    {
        const uint16_t* const k = in.k + t.row0 * in.k_ts + head * in.k_hs + ((uint32_t)tid / CPR * in.k_ts + tid % CPR * 8);
        const uint16_t* const v = in.v + t.row0 * in.v_ts + head * in.v_hs + ((uint32_t)tid / CPR * in.v_ts + tid % CPR * 8);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (tid + 256 * i < nt * CPR) {
                raw[0][i] = *reinterpret_cast<const u32x4*>(k + i * (kStep * in.k_ts));
                raw[1][i] = *reinterpret_cast<const u32x4*>(v + i * (kStep * in.v_ts));
            }
    }
    if (off < 0) return;                                            // (uniform)
    uint8_t* const blk = const_cast<uint8_t*>(p.pages) + off;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int ch = tid + 256 * i;
            if (ch >= nt * CPR) break;                              // (eight lanes of a group alike: CPR is a multiple of 8)
            const int tok = t.t0 + ch / CPR, d0 = ch % CPR * 8, g = d0 / kKv4Group;
            __builtin_assume(tok >= 0 && tok < 32);
            Enc en;
            encode_group<kBf16>(raw[which][i], en);
            // (the low 22 bits of lv are the level)
            if (which == 0) {
                const uint32_t even = en.lv[0] | en.lv[2] << 4 | en.lv[4] << 8 | en.lv[6] << 12;
                const uint32_t odd = en.lv[1] | en.lv[3] << 4 | en.lv[5] << 8 | en.lv[7] << 12;
                *reinterpret_cast<uint32_t*>(blk + kv4_k_word(HD, tok, d0)) = __builtin_amdgcn_perm(odd, even, 0x05040100u);
            } else {
                u32x2 bytes;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    bytes[w] = __builtin_amdgcn_perm(en.lv[4 * w + 1], en.lv[4 * w], 0x0C0C0400u) |
                               __builtin_amdgcn_perm(en.lv[4 * w + 3], en.lv[4 * w + 2], 0x04000C0Cu);
                *reinterpret_cast<u32x2*>(&lv[tok][d0]) = bytes;
            }
            if (tid % 8 == 0) {
                *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2 * which, tok, g)) = (uint16_t)st16<false>(en.s);
                *reinterpret_cast<uint16_t*>(blk + kv4_param(HD, 2 * which + 1, tok, g)) = (uint16_t)st16<false>(en.m);
            }
        }
    __syncthreads();
    // words of four dimensions d0 .. d0 + 3: tokens 4 h + r and 16 + 4 h + r
    for (int i = tid; i < HD; i += 256) {
        const int h = i / (HD / 4), d0 = i % (HD / 4) * 4;
        uint32_t b[8], fresh = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = e / 4 * 16 + 4 * h + e % 4;
            b[e] = *reinterpret_cast<const uint32_t*>(&lv[tok][d0]) & 0x0F0F0F0Fu;     // (old tokens' bytes were never set)
            if (tok >= t.t0 && tok < t.t1) fresh |= 15u << kv4_shift(e);
        }
        if (fresh == 0) continue;
        // bytes of four dimensions with the levels of two tokens each; byte j of a word is byte d of c[j]
        const uint32_t c[4] = {b[0] | b[2] << 4, b[4] | b[6] << 4, b[1] | b[3] << 4, b[5] | b[7] << 4};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const uint32_t word = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u + 0x0101u * d),
                                                        __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u + 0x0101u * d), 0x05040100u);
            uint32_t* const at = reinterpret_cast<uint32_t*>(blk + kv4_v_word(HD, 4 * h, d0 + d));
            *at = fresh == 0xFFFFFFFFu ? word : (*at & ~fresh) | (word & fresh);
        }
    }
}

// ---- read --------------------------------------------------------------------------------------
// The same cut: a work-group takes one block of one head into LDS (coalesced) and writes its new tokens' rows, K by
// words (eight dimensions of a token), V by four words side by side (eight tokens of four dimensions).  13081 rows of
// 8 heads of 128 in 13.3 us (69 MB, 5.2 TB/s).
struct RowsOut {
    uint16_t* k;
    uint16_t* v;
    int64_t k_ts, k_hs, v_ts, v_hs;
};

template <int HD, bool kBf16>
__global__ __launch_bounds__(256) void k_kv4_read(const Kv4Pool p, const RowsOut out) {
    constexpr int kBB = kv4_block_bytes(HD), CPR = HD / 8;
    __shared__ __align__(16) uint8_t blk[kBB];
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    Touched t;
    if (!find_touched(p, blockIdx.x, pre, &t)) return;
    const int head = blockIdx.y, tid = threadIdx.x;
    const int64_t off = block_offset(p, t.slot, head, t.block, kBB);
    for (int i = tid; i < kBB / 16; i += 256)
        reinterpret_cast<u32x4*>(blk)[i] = off < 0 ? u32x4{0u, 0u, 0u, 0u} : reinterpret_cast<const u32x4*>(p.pages + off)[i];
    __syncthreads();
    const int nt = t.t1 - t.t0;
    auto value = [](uint32_t level, float s, float m) { return __builtin_fmaf((float)(int)level, s, m); };
    for (int i = tid; i < nt * CPR; i += 256) {
        const int tok = t.t0 + i / CPR, d0 = i % CPR * 8, g = d0 / kKv4Group;
        const float s = sx8_h2f(*reinterpret_cast<const uint16_t*>(blk + kv4_param(HD, 0, tok, g)));
        const float m = sx8_h2f(*reinterpret_cast<const uint16_t*>(blk + kv4_param(HD, 1, tok, g)));
        const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + kv4_k_word(HD, tok, d0));
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = pack16<kBf16>(value(word >> kv4_shift(2 * e) & 15u, s, m), value(word >> kv4_shift(2 * e + 1) & 15u, s, m));
        *reinterpret_cast<u32x4*>(out.k + (int64_t)(t.row0 + i / CPR) * out.k_ts + head * out.k_hs + d0) = w;
    }
    for (int i = tid; i < HD; i += 256) {
        const int h = i / (HD / 4), d0 = i % (HD / 4) * 4, g = d0 / kKv4Group;
        uint32_t words[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) words[e] = *reinterpret_cast<const uint32_t*>(blk + kv4_v_word(HD, 4 * h, d0 + e));
        const u32x4 s8 = *reinterpret_cast<const u32x4*>(blk + kv4_param(HD, 2, 4 * h, g));
        const u32x4 m8 = *reinterpret_cast<const u32x4*>(blk + kv4_param(HD, 3, 4 * h, g));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int tok = e / 4 * 16 + 4 * h + e % 4;
            if (tok < t.t0 || tok >= t.t1) continue;
            const float s = sx8_h2f(half_of(s8[e >> 1], e)), m = sx8_h2f(half_of(m8[e >> 1], e));
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = value(words[k] >> kv4_shift(e) & 15u, s, m);
            *reinterpret_cast<u32x2*>(out.v + (int64_t)(t.row0 + tok - t.t0) * out.v_ts + head * out.v_hs + d0) =
                u32x2{pack16<kBf16>(x[0], x[1]), pack16<kBf16>(x[2], x[3])};
        }
    }
}

// ---- attend ------------------------------------------------------------------------------------
// The launch's waves share the blocks of all units evenly (sx8_kv4.h) and work apart from each other; a piece is a run
// of blocks of one unit.  Per block a wave computes S^T = K Q^T on v_mfma_f32_16x16x32_f16 with the tokens as
// rows and the unit's 16 query rows as columns, so that a lane (column c, step group h) holds the scores of
// tokens 4 h + r and 16 + 4 h + r of its own query row and the softmax stays in the lane.  The levels go into the
// MFMA as the fp16 subnormals level * 2^-20, which is a shift and a mask for two values and exact; the scale
// multiplies each group's 32-bit sum (q . k = sum_g s_g (q_g . level_g) + m_g sum(q_g)), and the minima's part is
// one more MFMA with sum(q_g) as two fp16 numbers.  O^T += V^T P^T takes the levels in the same way, with p * s of
// each token rounded to two fp16 numbers (22 bits), and the minima's part sum_t p_t m_t,g as MFMAs of their own.
// The MFMA aligns its products by their exponent fields, a subnormal's being 2^-14, and cuts what lies about 25 places below the
// largest: always downwards, so a sum of levels comes out too small by up to half a place a product.  As level * 2^-24 that
// is 2^-16 of a level, which many tokens do not average away while their values do (four slots of up to 131000 tokens: 5.5e-4
// of the outputs); as level * 2^-20 it is 2^-20 of one (1e-5 of them, the plain float32 form 4e-6).
// Query rows are multiplied by a power of two that brings their largest value into [64, 128), which is undone in
// the scale: rows become fp16 within 2^-31 of their largest value (exact where they hold nothing 2^-20 below it, bf16: 2^-23),
// and sum(q_g) fits.
// The running maximum is kept kUp powers of two below the largest score and raised when a score exceeds it by kUp + kSlack,
// so that p is at most 2^13, the largest weight at least 2^10, and p * s holds its 22 bits down to p * s = 2^-3 in those
// units (below that it is within 2^-25).  (Raised at every larger score, four long slots take 54.4 us instead of 51.7.)
// Scales of 2 or more (groups that span 30 or more) would take p * s out of fp16: those go in 2^k times smaller, below 2 and
// from 1/16 on, with their levels 2^k times as large, in matrix products of their own for each of k = 5, 10 and 15 that a
// block has.  So what is kept of a token does not depend on the scales of other groups or tokens.
// Bound by its chain of loads (lengths, table, block) first: a first block takes 6.2 us; then by memory and the VALU together: the
// blocks come at 4.3-5 TB/s, a stream that is only read at 6.1, with the VALU active 55% of the time (four long
// slots).  8 KV heads of 128: 48 slots of 60 .. 8000 tokens 21.7 us and the combine 4.0, 32 slots of 16384 tokens 122-139 us
// by machine.  Three sets of registers ahead instead of two: no faster.
template <int HD>
constexpr int waves_log2() { return HD == 256 ? 10 : 11; }        // one or two a SIMD of 256 CUs, as registers allow

// Record of a cut unit for the combine; parts == 0: none.  The records lie by unit (slots, heads, tiles) where the host
// knows that there are no more units than waves, so that the combine has a work-group for each; otherwise by the
// wave that has the unit's first block.
struct Kv4Piece {
    int32_t parts, first, tile, head, row0, n, pad[2];      // first: place of its first part
};
static_assert(sizeof(Kv4Piece) == 32, "record");

struct AttendIo {
    const uint16_t* q;
    uint16_t* out;
    int64_t q_ts, q_hs, o_ts, o_hs;
    float scale_log2;
    float* part_o;                        // [2 waves][16][HD]
    float* part_ml;                       // [2 waves][16][2]
    Kv4Piece* piece;                      // [waves]
    int by_unit;
};

constexpr int64_t attend_ws(int64_t hd) {
    return ((int64_t)(2 * 16 * (hd + 2) * 4 + sizeof(Kv4Piece))) << (hd == 256 ? 10 : 11);
}

// What a wave knows of the slots: with up to 64 of them lane s holds slot s and its place on the line of blocks; with
// more the places lie in LDS.
struct Slots {
    int row0, n, len;
    int64_t end;                          // places of the slots up to this lane's
    int units;                            // (by_unit) units of the slots up to this lane's
};

template <int HD, bool kBf16>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_kv4_attend(const Kv4Pool p, const AttendIo io) {
    using Regs = Kv4Regs<HD>;
    constexpr int W = Regs::W, NT = Regs::NT, NG = Regs::NG, kBB = kv4_block_bytes(HD);
    constexpr float kInf = __builtin_inff();
    int64_t* const pre = reinterpret_cast<int64_t*>(dyn_lds);
    const int lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int S = p.sh.n_slots, G = p.sh.G;
    const bool few = S <= 64;
    Slots sl = {0, 0, 0, 0, 0};
    int32_t* const pre_units = reinterpret_cast<int32_t*>(pre + S + 1);
    int64_t total;
    int units = 0;
    if (few) {
        if (lane < S) {
            kv4_rows(p.sh, p.cu, lane, &sl.row0, &sl.n);
            sl.len = kv4_len(p.sh, p.lens, lane);
            sl.end = kv4_slot_places(p.sh.nk, G, sl.n, sl.len);
            sl.units = p.sh.nk * kv4_tiles(sl.n, G);
        }
        sl.end = wave_prefix(sl.end);
        total = lane_of(sl.end, 63);
        if (io.by_unit) {
            sl.units = (int)wave_prefix(sl.units);
            units = __builtin_amdgcn_readlane(sl.units, 63);
        }
    } else {
        prefix_sums<256>(S, pre, [&](int s) { return kv4_slot_places(p.sh, p.lens, p.cu, s); });
        if (io.by_unit)
            prefix_sums<256>(S, pre_units, [&](int s) {
                int first, n;
                kv4_rows(p.sh, p.cu, s, &first, &n);
                return (int64_t)p.sh.nk * kv4_tiles(n, G);
            });
        __syncthreads();
        total = uniform(pre[S]);
        if (io.by_unit) units = __builtin_amdgcn_readfirstlane(pre_units[S]);
    }
    const int64_t share = kv4_share(total, waves_log2<HD>());
    const int64_t x0 = wave * share, x1 = x0 + share < total ? x0 + share : total;
    int slot = 0;
    if (x0 < total) {
        if (few) slot = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < S && sl.end <= x0));
        else
            for (int s = lane; s - lane < S; s += 64) slot += __builtin_popcountll(__builtin_amdgcn_ballot_w64(s < S && pre[s < S ? s + 1 : S] <= x0));
    }
    if ((!io.by_unit || wave >= units) && lane == 0) io.piece[wave].parts = 0;
    for (int64_t x = x0; x < x1;) {
        int row0, n, len;
        int64_t begin;
        int unit0 = 0;
        if (few) {
            while (x >= lane_of(sl.end, slot)) ++slot;
            row0 = __builtin_amdgcn_readlane(sl.row0, slot);
            n = __builtin_amdgcn_readlane(sl.n, slot);
            len = __builtin_amdgcn_readlane(sl.len, slot);
            begin = slot ? lane_of(sl.end, slot - 1) : 0;
            if (io.by_unit) unit0 = slot ? __builtin_amdgcn_readlane(sl.units, slot - 1) : 0;
        } else {
            while (x >= uniform(pre[slot + 1])) ++slot;
            kv4_rows(p.sh, p.cu, slot, &row0, &n);
            row0 = __builtin_amdgcn_readfirstlane(row0);
            n = __builtin_amdgcn_readfirstlane(n);
            len = __builtin_amdgcn_readfirstlane(kv4_len(p.sh, p.lens, slot));
            begin = uniform(pre[slot]);
            if (io.by_unit) unit0 = __builtin_amdgcn_readfirstlane(pre_units[slot]);
        }
        const int nb = kv4_unit_blocks(len), tiles = kv4_tiles(n, G);
        const Kv4Run run = kv4_run(x, x - begin, x1, nb);
        const int b0 = run.b0, bend = run.b1;
        const int64_t here = x;
        x += run.places;
        if (b0 == bend) continue;
        const int head = (int)kv4_div(run.unit, tiles), tile = (int)(run.unit - (int64_t)head * tiles);
        // the column's query row, and the last position it may attend
        const int r = 16 * tile + c, tok = r / G;
        const bool row_ok = tok < n;
        const int lim = row_ok ? len - n + tok : len - 1;
        const int tok_min = 16 * tile / G, tok_max = (16 * tile + 15) / G;
        const int lim_min = len - n + tok_min, lim_max = len - n + (tok_max < n ? tok_max : n - 1);
        const int b1 = lim_max < 0 ? b0 : bend < lim_max / 32 + 1 ? bend : lim_max / 32 + 1;   // blocks it reads
        const int cnt = b1 > b0 ? b1 - b0 : 0;
        int pages = -1;                                                    // lane i: page of block b0 + i0 + i
        auto load_pages = [&](int i0) {
            const int b = b0 + i0 + lane;
            pages = b < b1 ? p.table[(int64_t)slot * p.max_pages + (b >> p.bpp_log2)] : -1;
        };
        auto load = [&](Regs& rg, int i) __attribute__((always_inline)) {
            if (i != 0 && (i & 63) == 0) load_pages(i);
            const int b = b0 + i;
            int page = __builtin_amdgcn_readlane(pages, i & 63);
            rg.bad = page < 0 || page >= p.n_pages;
            page = rg.bad ? 0 : page;
            const uint8_t* base = p.pages + page * p.page_bytes
                + (int64_t)((head << p.bpp_log2) + (b & ((1 << p.bpp_log2) - 1))) * kBB;
            load_block<HD>(rg, base, lane);
        };
        load_pages(0);
        // query fragment: fp16 with the row's largest value in [64, 128)
        u32x4 raw[W];
        {
            const int tk = row_ok ? tok : 0, hd = head * G + (row_ok ? r - tok * G : 0);
            const uint16_t* qr = io.q + ((int64_t)row0 + tk) * io.q_ts + hd * io.q_hs + 8 * h;
#pragma unroll
            for (int j = 0; j < W; ++j) raw[j] = *reinterpret_cast<const u32x4*>(qr + 32 * j);
        }
        Regs r0, r1;
        if (cnt > 0) load(r0, 0);
        f16x8 qf[W], qm;
        float kscale;
        {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(ld16<kBf16>(half_of(raw[j][e >> 1], e))));
            top = max4(row_ok ? top : 0.f);
            // exponent of the largest value; no scaling of rows that are zero or not finite
            const int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
            const int up = top > 0.f && ex < 255 && ex > 0 ? (127 + 6 - ex < 126 ? 127 + 6 - ex : 126) : 0;
            const float mul = __builtin_ldexpf(row_ok ? 1.f : 0.f, up);
            kscale = io.scale_log2 * __builtin_ldexpf(1.f, -up);
            float qs[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) qs[g] = 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float raw_q = ld16<kBf16>(half_of(raw[j][e >> 1], e));
                    const _Float16 v = (_Float16)(row_ok ? raw_q * mul : 0.f);
                    qf[j][e] = v;
                    qs[j / 2] += (float)v;
                }
#pragma unroll
            for (int e = 0; e < 8; ++e) qm[e] = (_Float16)0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float s = sum4(qs[g]);
                const _Float16 hi = (_Float16)s;
                if (h == 0) {
                    qm[g] = hi;
                    qm[4 + g] = (_Float16)(s - (float)hi);
                }
            }
        }
        f32x4 o[NT], om = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -kInf, l = 0.f;
        auto step = [&](Regs& rg, int i) __attribute__((always_inline)) {
            const int b = b0 + i;
            const bool mask = b * 32 + 31 > lim_min || rg.bad;     // past a column's last position, or no page
            float sc[8];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                    acc = mfma16(levels(rg.kw[a][2 * g]), qf[2 * g], acc);
                    acc = mfma16(levels(rg.kw[a][2 * g + 1]), qf[2 * g + 1], acc);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[e] = __builtin_fmaf(sx8_h2f(half_of(rg.ks[g][2 * a + (e >> 1)], e)), acc[e], s[e]);
                }
                u32x4 mw = {0u, 0u, 0u, 0u};
                if (h == 0) {
                    mw.x = rg.km[a][0];
                    mw.z = rg.km[a][0];
                    if constexpr (NG == 4) mw.y = mw.w = rg.km[a][1];
                }
                const f32x4 mt = mfma16(__builtin_bit_cast(f16x8, mw), qm, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[4 * a + e] = __builtin_fmaf(s[e], 1048576.f, mt[e]);
            }
            if (mask) {
                asm volatile("");                // (a branch: as selects these would run for every block)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = b * 32 + (e / 4) * 16 + 4 * h + e % 4;
                    sc[e] = key <= lim && !rg.bad ? sc[e] : -kInf;
                }
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
            mx *= kscale;
            if (__builtin_amdgcn_ballot_w64(mx > m + (kUp + kSlack)) != 0) {
                const float mn = fmaxf(m, max4(mx - kUp));
                const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= alpha;
                om *= alpha;
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t] *= alpha;
            }
            const float nm = m == -kInf ? 0.f : -m;
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], kscale, nm));
                l += pv[e];
            }
            u32x4 vm = rg.vm;
            if (c >= NG) vm = u32x4{0u, 0u, 0u, 0u};
            if (mask) {
                // a token that some column may not attend must not reach it through 0 * NaN: its scale is zero for that
                // column, and its minimum zero where it is no number (the scale, which is none either, still brings the
                // NaN to the columns that attend it, however small its weight)
                asm volatile("");
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = b * 32 + (e / 4) * 16 + 4 * h + e % 4;
                    if (key > lim || rg.bad)
#pragma unroll
                        for (int g = 0; g < NG; ++g) rg.vs[g][e >> 1] &= e & 1 ? 0xFFFFu : 0xFFFF0000u;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = vm[e] & 0x7FFFu, hi = vm[e] >> 16 & 0x7FFFu;
                    vm[e] = (lo >= 0x7C00u ? 0u : vm[e] & 0xFFFFu) | (hi >= 0x7C00u ? 0u : vm[e] & 0xFFFF0000u);
                }
            }
            u32x4 ph, pl;
            constexpr uint32_t kOnes = 0x3C003C00u;
            split8(pv, u32x4{kOnes, kOnes, kOnes, kOnes}, &ph, &pl);
            const f16x8 vm8 = __builtin_bit_cast(f16x8, vm);
            om = mfma16(vm8, __builtin_bit_cast(f16x8, ph), om);
            om = mfma16(vm8, __builtin_bit_cast(f16x8, pl), om);
            uint32_t large = 0;                  // bits 14 and 30: a scale of 2 or more (or NaN)
#pragma unroll
            for (int g = 0; g < NG; ++g) large |= rg.vs[g][0] | rg.vs[g][1] | rg.vs[g][2] | rg.vs[g][3];
            if (__builtin_amdgcn_ballot_w64((large & 0x40004000u) != 0) != 0) {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll 1
                    for (int k = 5; k <= 15; k += 5) {
                        u32x4 s = large_scales(rg.vs[g], k);
                        if (__builtin_amdgcn_ballot_w64((s[0] | s[1] | s[2] | s[3]) != 0) == 0) continue;
                        const _Float16 down = (_Float16)__builtin_ldexpf(1.f, -k), up = (_Float16)__builtin_ldexpf(1.f, k);
                        s = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, s) * f16x8(down));
                        u32x4 hi, lo;
                        split8(pv, s, &hi, &lo);
#pragma unroll
                        for (int t = 4 * g; t < 4 * g + 4; ++t) {
                            uint32_t w = rg.vw[t];
                            asm volatile("" : "+v"(w));          // (here, not ahead of the loop: registers)
                            const f16x8 lv = levels(w) * f16x8(up);
                            o[t] = mfma16(lv, __builtin_bit_cast(f16x8, hi), o[t]);
                            o[t] = mfma16(lv, __builtin_bit_cast(f16x8, lo), o[t]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) rg.vs[g][e] &= ~((rg.vs[g][e] >> 14 & 0x00010001u) * 0xFFFFu);
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                u32x4 hi, lo;
                split8(pv, rg.vs[g], &hi, &lo);
                const f16x8 h8 = __builtin_bit_cast(f16x8, hi), l8 = __builtin_bit_cast(f16x8, lo);
#pragma unroll
                for (int t = 4 * g; t < 4 * g + 4; ++t) {
                    const f16x8 lv = levels(rg.vw[t]);
                    o[t] = mfma16(lv, h8, o[t]);
                    o[t] = mfma16(lv, l8, o[t]);
                }
            }
        };
        for (int i = 0; i < cnt; i += 2) {
            if (i + 1 < cnt) load(r1, i + 1);
            step(r0, i);
            if (i + 1 >= cnt) break;
            if (i + 2 < cnt) load(r0, i + 2);
            step(r1, i + 1);
        }
        // O = 2^20 (levels) + (the minima's sum of the group, row g of om)
        l = sum4(l);
        const bool whole = b0 == 0 && bend == nb;
        const float f = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const int place = 2 * wave + (here == x0 ? 0 : 1);
        const int64_t at = place * (int64_t)16 + c;
        float* const po = io.part_o + at * HD + 4 * h;
        uint16_t* const dst = io.out + ((int64_t)row0 + tok) * io.o_ts + (head * G + (r - tok * G)) * io.o_hs + 4 * h;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float og = __shfl(om[t / 4], c, 64);
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[t][e], 1048576.f, og) * f;
            if (row_ok) {
                if (whole) *reinterpret_cast<u32x2*>(dst + 16 * t) = u32x2{pack16<kBf16>(v[0], v[1]), pack16<kBf16>(v[2], v[3])};
                else *reinterpret_cast<f32x4*>(po + 16 * t) = v;
            }
        }
        if (!whole && h == 0 && row_ok) {
            io.part_ml[at * 2] = m;
            io.part_ml[at * 2 + 1] = l;
        }
        // the unit's record is written by its first piece; a unit that is cut goes on in the next waves
        // (a cu that runs backwards can name more units than rows allow: those have no record)
        const int64_t rec = io.by_unit ? unit0 + run.unit : wave;
        if (b0 == 0 && lane == 0 && (io.by_unit || !whole) && rec < (1 << waves_log2<HD>())) {
            Kv4Piece pc;
            pc.parts = whole ? 0 : kv4_parts(begin + run.unit * (nb + kKv4Begin) + kKv4Begin, nb, share, wave);
            pc.first = place;
            pc.tile = tile;
            pc.head = head;
            pc.row0 = row0;
            pc.n = n;
            io.piece[rec] = pc;
        }
    }
}

// Units that were cut: work-group (i, row) takes a row of record i and adds the unit's parts up in their order (part 0 at its
// place, part j at place 2 (wave + j)).  The parts are shared by kWaves waves, whose sums meet in LDS.  A launch costs 1.8
// us and three dependent loads; 48 slots of up to 8000 tokens take 4.0-4.7 us, 16 slots of 8 new tokens 5.6-6.0 (work-groups of
// 16 waves for four rows at once: 5.9 and 6.5; two waves a row: 4.8 and 5.1, but twice the rounds where one slot of
// many has most of the tokens).
template <int HD, bool kBf16, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void k_kv4_combine(const AttendIo io, int G) {
    constexpr int N = HD / 64, kU = 8;                            // kU: parts requested together
    typedef float vecN __attribute__((ext_vector_type(N)));
    const Kv4Piece pc = io.piece[blockIdx.x];
    const int row = blockIdx.y;
    if (pc.parts == 0 || row >= min(16, pc.n * G - 16 * pc.tile)) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ float sml[kWaves][2];
    __shared__ vecN so[kWaves][64];
    auto at = [&](int i) { return (int64_t)(i == 0 ? pc.first : 2 * (pc.first / 2 + i)) * 16 + row; };
    const int per = (pc.parts + kWaves - 1) / kWaves, i0 = w * per, i1 = min(i0 + per, pc.parts);
    float m = -__builtin_inff(), den = 0.f;
    vecN acc = 0.f;
    for (int i = i0; i < i1; i += kU) {
        float pm[kU], pl[kU];
        vecN v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int64_t a = at(min(i + u, i1 - 1));
            pm[u] = io.part_ml[a * 2];
            pl[u] = io.part_ml[a * 2 + 1];
            v[u] = reinterpret_cast<const vecN*>(io.part_o + a * HD)[lane];
        }
        __builtin_amdgcn_sched_barrier(0);
        float mn = m;
#pragma unroll
        for (int u = 0; u < kU; ++u) mn = fmaxf(mn, pm[u]);
        const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        den *= alpha;
        acc *= alpha;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (i + u >= i1) continue;
            const float f = pm[u] == m ? 1.f : __builtin_amdgcn_exp2f(pm[u] - m);
            den = __builtin_fmaf(f, pl[u], den);
            acc = __builtin_elementwise_fma(vecN(f), v[u], acc);
        }
    }
    if (lane == 0) {
        sml[w][0] = m;
        sml[w][1] = den;
    }
    so[w][lane] = acc;
    __syncthreads();
    if (w != 0) return;
    float mm = m;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) mm = fmaxf(mm, sml[i][0]);
    const float f0 = m == mm ? 1.f : __builtin_amdgcn_exp2f(m - mm);
    den *= f0;
    acc *= f0;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        const float f = sml[i][0] == mm ? 1.f : __builtin_amdgcn_exp2f(sml[i][0] - mm);
        den = __builtin_fmaf(f, sml[i][1], den);
        acc = __builtin_elementwise_fma(vecN(f), so[i][lane], acc);
    }
    acc *= den == 0.f ? 0.f : 1.f / den;
    const int rr = 16 * pc.tile + row, tk = rr / G;
    uint16_t* dst = io.out + ((int64_t)pc.row0 + tk) * io.o_ts + (pc.head * G + (rr - tk * G)) * io.o_hs + N * lane;
    if constexpr (N == 1) *dst = (uint16_t)st16<kBf16>(acc[0]);
    else
#pragma unroll
        for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack16<kBf16>(acc[e], acc[e + 1]);
}

}  // namespace
}  // namespace sx8

extern "C" int64_t sx8_kv4_page_bytes(int32_t nk, int32_t hd, int32_t page_tokens) {
    using namespace sx8;
    if (nk < 1 || nk > 256 || !hd_ok(hd) || (page_tokens != 32 && page_tokens != 64 && page_tokens != 128 && page_tokens != 256))
        return -1;
    return (int64_t)nk * (page_tokens / 32) * kv4_block_bytes(hd);
}

extern "C" int32_t sx8_kv4_append(uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                  int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* k, const void* v,
                                  int64_t rows, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, int32_t nk,
                                  int32_t hd, int32_t page_tokens, int32_t dtype, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_append";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "k", k, k_ts, k_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "v", v, v_ts, v_hs, rows);
    if (rc != SX8_OK) return rc;
    if (rows == 0) return ok();
    const RowsIn in{(const uint16_t*)k, (const uint16_t*)v, k_ts, k_hs, v_ts, v_hs};
    const dim3 grid((unsigned)kv4_touched_most(n_slots, rows, cu != nullptr), (unsigned)nk);
    by_kind(hd, dtype, [&](auto d, auto b) {
        hipLaunchKernelGGL((k_kv4_append<decltype(d)::value, decltype(b)::value>), grid, dim3(256),
                           cu && n_slots > 64 ? prefix_bytes(p) : 0, as_stream(stream), p, in);
    });
    return check_launch(what);
}

extern "C" int32_t sx8_kv4_read(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                int64_t n_slots, int64_t max_pages, int64_t n_pages, void* k, void* v, int64_t rows,
                                int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, int32_t nk, int32_t hd,
                                int32_t page_tokens, int32_t dtype, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_read";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "k", k, k_ts, k_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "v", v, v_ts, v_hs, rows);
    if (rc == SX8_OK) rc = check_apart(what, "k", k_ts, k_hs, rows, nk, hd);
    if (rc == SX8_OK) rc = check_apart(what, "v", v_ts, v_hs, rows, nk, hd);
    if (rc != SX8_OK) return rc;
    if (rows == 0) return ok();
    const RowsOut out{(uint16_t*)k, (uint16_t*)v, k_ts, k_hs, v_ts, v_hs};
    const dim3 grid((unsigned)kv4_touched_most(n_slots, rows, cu != nullptr), (unsigned)nk);
    by_kind(hd, dtype, [&](auto d, auto b) {
        hipLaunchKernelGGL((k_kv4_read<decltype(d)::value, decltype(b)::value>), grid, dim3(256),
                           cu && n_slots > 64 ? prefix_bytes(p) : 0, as_stream(stream), p, out);
    });
    return check_launch(what);
}

extern "C" int64_t sx8_kv4_attend_workspace_bytes(int32_t hd) { return sx8::hd_ok(hd) ? sx8::attend_ws(hd) : -1; }

extern "C" int32_t sx8_kv4_attend(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                                  int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* q, void* out,
                                  int64_t rows, int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs, int32_t nh,
                                  int32_t nk, int32_t hd, int32_t page_tokens, float scale, int32_t dtype,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_attend";
    Kv4Pool p;
    int32_t rc = make_pool(what, &p, pages, table, lens, cu, n_slots, max_pages, n_pages, rows, nk, hd, page_tokens, dtype);
    if (rc == SX8_OK) rc = check_rows(what, "q", q, q_ts, q_hs, rows);
    if (rc == SX8_OK) rc = check_rows(what, "out", out, o_ts, o_hs, rows);
    if (rc != SX8_OK) return rc;
    if (nh <= 0 || nh % nk || nh / nk > 256)
        return fail(SX8_ERR_INVALID, "%s: nh must be a multiple of nk, at most 256 nk", what);
    rc = check_apart(what, "out", o_ts, o_hs, rows, nh, hd);
    if (rc != SX8_OK) return rc;
    if (!(scale > 0.f) || !(scale < __builtin_inff()))
        return fail(SX8_ERR_INVALID, "%s: scale must be positive and finite", what);
    if (!workspace || workspace_bytes < attend_ws(hd) || !aligned(workspace, 256))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 256-byte aligned", what, (long long)attend_ws(hd));
    if (rows * (nh / nk) > 0x7FFFFF00) return fail(SX8_ERR_UNSUPPORTED, "%s: over 2^31 query rows of a KV head", what);
    if (rows == 0) return ok();
    p.sh.G = nh / nk;
    const int64_t waves = (int64_t)1 << (hd == 256 ? 10 : 11);
    AttendIo io{(const uint16_t*)q, (uint16_t*)out, q_ts, q_hs, o_ts, o_hs, scale * 1.4426950408889634f, nullptr, nullptr,
                nullptr, 0};
    io.piece = reinterpret_cast<Kv4Piece*>(workspace);
    io.part_o = reinterpret_cast<float*>(io.piece + waves);
    io.part_ml = io.part_o + 2 * waves * 16 * hd;
    // units at most: a slot with n rows has nk ceil(n G / 16) of them
    const int64_t G = p.sh.G, live = n_slots < rows ? n_slots : rows;
    const int64_t units = nk * (cu ? rows * G / 16 + live : n_slots * ((G + 15) / 16));
    io.by_unit = units <= waves;
    const unsigned entries = (unsigned)(io.by_unit ? units : waves), used = (unsigned)(cu ? (rows * G < 16 ? rows * G : 16) : (G < 16 ? G : 16));
    // few rows in all: a row's parts are shared by 16 waves, else by four
    const bool narrow = entries * used <= 512;
    by_kind(hd, dtype, [&](auto d, auto b) {
        constexpr int HD = decltype(d)::value;
        constexpr bool kBf = decltype(b)::value;
        hipLaunchKernelGGL((k_kv4_attend<HD, kBf>), dim3((1 << waves_log2<HD>()) / 4), dim3(256),
                           n_slots <= 64 ? 0 : prefix_bytes(p) * 3 / 2, as_stream(stream), p, io);
        const dim3 grid(entries, used);
        if (narrow) hipLaunchKernelGGL((k_kv4_combine<HD, kBf, 16>), grid, dim3(1024), 0, as_stream(stream), io, p.sh.G);
        else hipLaunchKernelGGL((k_kv4_combine<HD, kBf, 4>), grid, dim3(256), 0, as_stream(stream), io, p.sh.G);
    });
    return check_launch(what);
}
