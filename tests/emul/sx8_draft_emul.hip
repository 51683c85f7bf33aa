// Host build of the tree attention's masks and work split (sx8-quantization_amd/csrc/sx8_kv4.h), the functions the kernel
// calls.  Built host-only by tests/test_draft_cpu.py; never loaded on the GPU path.
#include "sx8_kv4.h"

using namespace sx8;

extern "C" uint32_t sx8e_tree_bits(const uint64_t* mask, int32_t words, int32_t first, int32_t key0) {
    return kv4_tree_bits(mask, words, first, key0);
}

// The pieces of every work-group, as the attention walks them: (group, slot, unit of the slot, first block, end, blocks of the
// unit, place, parts, whole).
extern "C" int64_t sx8e_tree_pieces(int32_t n_slots, int32_t nk, int32_t G, int32_t cap, int32_t rows, int32_t cols,
                                    const int32_t* lens, const int32_t* cu, int32_t groups, int64_t* out, int64_t most) {
    const Kv4Shape sh{n_slots, nk, G, cap, rows};
    auto places = [&](int s) {
        int first, n;
        kv4_rows(sh, cu, s, &first, &n);
        return kv4_tree_places(sh, cols, n, kv4_len(sh, lens, s));
    };
    int64_t total = 0, got = 0;
    for (int s = 0; s < n_slots; ++s) total += places(s);
    const int64_t share = kv4_tree_share(total, groups);
    for (int64_t g = 0; g < groups; ++g) {
        const int64_t x0 = g * share, x1 = x0 + share < total ? x0 + share : total;
        int64_t before = 0;
        int s = 0;
        for (int64_t x = x0; x < x1;) {
            while (x >= before + places(s)) before += places(s++);
            const int nb = kv4_unit_blocks(kv4_len(sh, lens, s));
            const Kv4Run r = kv4_run(x, x - before, x1, nb, kTreeBegin);
            if (r.b0 != r.b1) {
                if (got < most) {
                    const bool whole = r.b0 == 0 && r.b1 == nb;
                    const int64_t v[9] = {g, s, r.unit, r.b0, r.b1, nb, 2 * g + (x != x0),
                                          (before + r.unit * (nb + kTreeBegin) + kTreeBegin + nb - 1) / share - g + 1, whole};
                    for (int i = 0; i < 9; ++i) out[got * 9 + i] = v[i];
                }
                ++got;
            }
            x += r.places;
        }
    }
    return got;
}
