// sx8_kv4.h -- the 4-bit KV cache format: where a value's bits lie, and how the attention over it is
// cut into pieces.  Plain integer functions, the same on the host (tests) and in the kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define SX8_KV4_FN __host__ __device__ __forceinline__

namespace sx8 {

constexpr int kKv4Group = 64;        // values that share a scale and a minimum
constexpr int kKv4Block = 32;        // tokens of a block
constexpr int kKv4MaxSlots = 4096;
constexpr int64_t kKv4MaxTokens = 1 << 22;   // of a slot (max_pages * page_tokens)

// A block holds the K and V rows of 32 tokens of one head:
//   K levels (16 hd bytes) | V levels (16 hd) | K scales | K minima | V scales | V minima (hd / 64 * 64 each)
// Levels are 4-bit, eight to a 32-bit word (value e of a word at bits 4 (e / 2) + 16 (e % 2), so that
// (word >> 4 i) & 0x000F000F are values 2 i and 2 i + 1 as two 16-bit numbers), and lie as a 16x16x32 MFMA
// takes them as its row operand: lane 16 h + c of 64 holds row c, steps 8 h .. 8 h + 7.
//   K: rows are tokens (two tiles of 16), steps are dimensions: word j of a lane covers dimensions 32 j + 8 h + e.
//   V: rows are dimensions (tile t: 16 t + c), steps are tokens: value e of the word of a lane is token
//      16 (e / 4) + 4 h + e % 4 -- the order in which the score tiles' accumulators hold them.
SX8_KV4_FN constexpr int kv4_block_bytes(int hd) { return 32 * hd + hd / kKv4Group * 256; }
SX8_KV4_FN constexpr int kv4_shift(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

// Byte offset in the block of the word that holds dimension d of token t, and the bit it starts at.
SX8_KV4_FN uint32_t kv4_k_word(uint32_t hd, uint32_t t, uint32_t d) {
    const uint32_t W = hd / 32, wi = W < 4 ? W : 4, j = d / 32, lane = (d % 32) / 8 * 16 + t % 16;
    return t / 16 * (256 * W) + (j / wi * 64 + lane) * wi * 4 + j % wi * 4;
}
SX8_KV4_FN int kv4_k_shift(int d) { return kv4_shift(d % 8); }
SX8_KV4_FN uint32_t kv4_v_word(uint32_t hd, uint32_t t, uint32_t d) {
    const uint32_t lane = (t % 16) / 4 * 16 + d % 16, tile = d / 16;
    return 16 * hd + (tile / 4 * 64 + lane) * 16 + tile % 4 * 4;
}
SX8_KV4_FN int kv4_v_shift(int t) { return kv4_shift(t / 16 * 4 + t % 4); }

// Scales of K (which = 0) and V (2) and minima of V (3) by group, step group h and token slot; minima of K (1)
// by token and group.
SX8_KV4_FN uint32_t kv4_param(uint32_t hd, uint32_t which, uint32_t t, uint32_t g) {
    const uint32_t ng = hd / kKv4Group, base = 32 * hd + which * ng * 64;
    return which == 1 ? base + 2 * (t * ng + g) : base + 2 * (g * 32 + (t % 16) / 4 * 8 + t / 16 * 4 + t % 4);
}

// ---- the attention's pieces -------------------------------------------------------------------
// A unit is 16 query rows (row r = token r / G, head r % G of the group) of one KV head of a slot; it reads the
// slot's blocks.  Units lie one after another (slots, heads, row tiles) on a line that the waves of the launch share
// evenly, so a unit may be cut into several pieces, each a run of blocks.  On the line a unit is its blocks and kKv4Begin
// places before them, for what a piece costs beside its blocks (a wave that gets only those has nothing to do).  With 1,
// 3 and 6 of them 48 slots of 60 .. 8000 tokens take 27.3, 25.0 and 24.7 us, 16 slots of 8 new tokens 20.5, 19.2 and 19.5.
constexpr int kKv4Begin = 3;
struct Kv4Shape {
    int n_slots, nk, G;
    int cap, rows;                 // tokens a slot can hold; query rows in the call (rows * G < 2^31)
};

// New tokens of slot s and the row of its first one, from cu (null: one row a slot), kept inside the call's rows.
SX8_KV4_FN int kv4_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
SX8_KV4_FN void kv4_rows(const Kv4Shape& sh, const int32_t* cu, int s, int* first, int* n) {
    const int a = kv4_clamp(cu ? cu[s] : s, 0, sh.rows), b = kv4_clamp(cu ? cu[s + 1] : s + 1, a, sh.rows);
    *first = a;
    *n = b - a;
}
SX8_KV4_FN int kv4_len(const Kv4Shape& sh, const int32_t* lens, int s) { return kv4_clamp(lens[s], 0, sh.cap); }
SX8_KV4_FN int kv4_unit_blocks(int len) { return len > 0 ? (len + kKv4Block - 1) / kKv4Block : 1; }
SX8_KV4_FN int kv4_tiles(int n, int G) { return (n * G + 15) / 16; }
// Places of a slot on the line.
SX8_KV4_FN int64_t kv4_slot_places(int nk, int G, int n, int len) {
    return (int64_t)nk * kv4_tiles(n, G) * (kv4_unit_blocks(len) + kKv4Begin);
}
SX8_KV4_FN int64_t kv4_slot_places(const Kv4Shape& sh, const int32_t* lens, const int32_t* cu, int s) {
    int first, n;
    kv4_rows(sh, cu, s, &first, &n);
    return kv4_slot_places(sh.nk, sh.G, n, kv4_len(sh, lens, s));
}

// Places of each of 2^waves_log2 waves: an even share.
SX8_KV4_FN int64_t kv4_share(int64_t total, int waves_log2) {
    const int64_t p = (total + (1 << waves_log2) - 1) >> waves_log2;
    return p < 1 ? 1 : p;
}
// The piece that begins at place x of the line, `off` places behind the beginning of its slot, for a wave whose share ends
// at x1: blocks b0 .. b1 - 1 of unit `unit` of the slot (none where b0 == b1), and the places it takes.
struct Kv4Run {
    int64_t unit;
    int b0, b1;
    int64_t places;
};
// a / b; the wide division only where it is needed
SX8_KV4_FN int64_t kv4_div(int64_t a, int b) { return (uint64_t)a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }
SX8_KV4_FN Kv4Run kv4_run(int64_t x, int64_t off, int64_t x1, int nb) {
    const int all = nb + kKv4Begin;
    const int64_t unit = kv4_div(off, all);
    const int v0 = (int)(off - unit * all), v1 = all - v0 < x1 - x ? all : v0 + (int)(x1 - x);
    return Kv4Run{unit, v0 > kKv4Begin ? v0 - kKv4Begin : 0, v1 > kKv4Begin ? v1 - kKv4Begin : 0, v1 - v0};
}
// How many waves have blocks of a unit whose first block lies at place `at`, in the share of `wave`.
SX8_KV4_FN int kv4_parts(int64_t at, int nb, int64_t share, int wave) {
    return (int)((at + nb - 1) / share - wave + 1);
}

// Blocks of tokens that the new tokens of a slot touch (append, read): first block, and how many.  Positions
// len - n .. len - 1; those below zero (more rows than tokens) lie in blocks below zero, which have no page.
SX8_KV4_FN int kv4_floor_block(int pos) { return pos >= 0 ? pos / kKv4Block : -((-pos + kKv4Block - 1) / kKv4Block); }
SX8_KV4_FN int kv4_touched(int len, int n, int* first) {
    *first = kv4_floor_block(len - n);
    return n > 0 ? kv4_floor_block(len - 1) - *first + 1 : 0;
}
// At least the touched blocks of all slots together, from what the host knows: every slot with rows touches at
// most (n + 30) / 32 + 1 blocks.
SX8_KV4_FN int64_t kv4_touched_most(int64_t n_slots, int64_t rows, bool cu) {
    return cu ? rows / kKv4Block + 2 * (n_slots < rows ? n_slots : rows) : (n_slots < rows ? n_slots : rows);
}

// Whether the head rows (hd values each) of a (rows, heads, hd) tensor lie apart from each other.
inline bool rows_apart(int64_t ts, int64_t hs, int64_t rows, int64_t heads, int64_t hd) {
    const bool by_rows = (hs >= hd || heads == 1) && (rows == 1 || ts >= (heads - 1) * hs + hd);
    return by_rows || ((ts >= hd || rows == 1) && (heads == 1 || hs >= (rows - 1) * ts + hd));
}

}  // namespace sx8
