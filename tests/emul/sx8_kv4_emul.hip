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

// The pieces of every wave, as the attention walks them: (wave, slot, unit of the slot, first block, end, blocks of
// the unit, place, parts), place = 2 wave + (0: the piece begins the share), parts (of a first piece) the waves that
// have blocks of the unit; at most `most` pieces, their number returned.
extern "C" int64_t sx8e_kv4_pieces(int32_t n_slots, int32_t nk, int32_t G, int32_t cap, int32_t rows, const int32_t* lens,
                                   const int32_t* cu, int32_t waves_log2, int64_t* out, int64_t most) {
    const Kv4Shape sh{n_slots, nk, G, cap, rows};
    int64_t total = 0, got = 0;
    for (int s = 0; s < n_slots; ++s) total += kv4_slot_places(sh, lens, cu, s);
    const int64_t share = kv4_share(total, waves_log2);
    for (int64_t w = 0; w < 1 << waves_log2; ++w) {
        const int64_t x0 = w * share, x1 = x0 + share < total ? x0 + share : total;
        int64_t before = 0;
        int s = 0;
        for (int64_t x = x0; x < x1;) {
            while (x >= before + kv4_slot_places(sh, lens, cu, s)) before += kv4_slot_places(sh, lens, cu, s++);
            const int nb = kv4_unit_blocks(kv4_len(sh, lens, s));
            const Kv4Run r = kv4_run(x, x - before, x1, nb);
            if (r.b0 != r.b1) {
                if (got < most) {
                    const int64_t at = before + r.unit * (nb + kKv4Begin) + kKv4Begin;
                    const int64_t v[8] = {w, s, r.unit, r.b0, r.b1, nb, 2 * w + (x != x0),
                                          r.b0 == 0 ? kv4_parts(at, nb, share, (int)w) : 0};
                    for (int i = 0; i < 8; ++i) out[got * 8 + i] = v[i];
                }
                ++got;
            }
            x += r.places;
        }
    }
    return got;
}
extern "C" int64_t sx8e_kv4_slot_places(int32_t n_slots, int32_t nk, int32_t G, int32_t cap, int32_t rows, const int32_t* lens,
                                        const int32_t* cu, int32_t s) {
    return kv4_slot_places(Kv4Shape{n_slots, nk, G, cap, rows}, lens, cu, s);
}
extern "C" int64_t sx8e_kv4_touched(int32_t len, int32_t n, int32_t* first) { return kv4_touched(len, n, first); }
extern "C" int64_t sx8e_kv4_touched_most(int64_t n_slots, int64_t rows, int32_t cu) {
    return kv4_touched_most(n_slots, rows, cu != 0);
}
