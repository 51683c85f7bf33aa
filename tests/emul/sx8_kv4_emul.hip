// Host build of the 4-bit cache's addressing and work split (sx8-quantization_amd/csrc/sx8_kv4.h), the functions the
// kernels call.  Built host-only by tests/test_kv4_cpu.py; never loaded on the GPU path.
#include "sx8_kv4.h"

using namespace sx8;

// where[0..3]: K word byte, K bit, V word byte, V bit of (t, d); then the four parameters' bytes of (t, d's group)
extern "C" void sx8e_kv4_where(int32_t hd, int32_t t, int32_t d, int32_t* where) {
    where[0] = kv4_k_word(hd, t, d);
    where[1] = kv4_k_shift(d);
    where[2] = kv4_v_word(hd, t, d);
    where[3] = kv4_v_shift(t);
    for (int i = 0; i < 4; ++i) where[4 + i] = kv4_param(hd, i, t, d / kKv4Group);
}
extern "C" int32_t sx8e_kv4_block_bytes(int32_t hd) { return kv4_block_bytes(hd); }

// The pieces of every work-group, as the attention walks them: (wg, slot, unit of the slot, first block, end, blocks of
// the unit, place), place = 2 wg + (0: the piece begins the share); at most `most` pieces, their number returned.
extern "C" int64_t sx8e_kv4_pieces(int32_t n_slots, int32_t nk, int32_t G, int64_t cap, int64_t rows, const int32_t* lens,
                                   const int32_t* cu, int32_t wgs, int64_t* out, int64_t most) {
    const Kv4Shape sh{n_slots, nk, G, cap, rows};
    int64_t total = 0, got = 0;
    for (int s = 0; s < n_slots; ++s) total += kv4_slot_blocks(sh, lens, cu, s);
    const int64_t share = kv4_share(total, wgs);
    for (int wg = 0; wg < wgs; ++wg) {
        const int64_t x0 = wg * share, x1 = x0 + share < total ? x0 + share : total;
        int64_t before = 0;
        int s = 0;
        for (int64_t x = x0; x < x1;) {
            while (x >= before + kv4_slot_blocks(sh, lens, cu, s)) before += kv4_slot_blocks(sh, lens, cu, s++);
            const int64_t nb = kv4_unit_blocks(kv4_len(sh, lens, s)), unit = (x - before) / nb, b0 = (x - before) % nb;
            const int64_t e = nb - b0 < x1 - x ? nb : b0 + (x1 - x);
            if (got < most) {
                const int64_t v[7] = {wg, s, unit, b0, e, nb, 2 * (int64_t)wg + (x != x0)};
                for (int i = 0; i < 7; ++i) out[got * 7 + i] = v[i];
            }
            ++got;
            x += e - b0;
        }
    }
    return got;
}
extern "C" int64_t sx8e_kv4_slot_blocks(int32_t n_slots, int32_t nk, int32_t G, int64_t cap, int64_t rows, const int32_t* lens,
                                        const int32_t* cu, int32_t s) {
    return kv4_slot_blocks(Kv4Shape{n_slots, nk, G, cap, rows}, lens, cu, s);
}
extern "C" int64_t sx8e_kv4_touched(int64_t len, int64_t n, int64_t* first) { return kv4_touched(len, n, first); }
extern "C" int64_t sx8e_kv4_touched_most(int64_t n_slots, int64_t rows, int32_t cu) {
    return kv4_touched_most(n_slots, rows, cu != 0);
}
