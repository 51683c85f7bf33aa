// sx8_pages.hip -- page operations of the paged KV cache: reserve, fork, free, compact and keep
// (include/sx8_paged.h).
//
// The tables are small and the decisions on them ordered (lowest free page first, all or nothing), so one work-group
// makes them; what moves bytes runs on the whole GPU behind it and reads its list of page pairs from the
// workspace.  Nothing depends on the order in which threads run: reference counts are integer sums.
// Decisions take 2.8 us (reserve, 24 slots) to 5.2 (fork, 64 entries), bound by their few dependent loads; the copies run
// at memory speed: compact moves 302 MB (read and written) in 47 us, 6.4 TB/s, 64 forks 76 MB in 10.6 us.
// keep decides in 4.4 us and moves the kept rows of 48 trees in eight layers in 12.5 (1.3 MB): a work-group takes a slot, head and layer,
// and its threads wait for the level of each token of a V word, up to eight of them, before they ask for the next one's.
#include "sx8_host.h"
#include "sx8_kv4_dev.h"
#include "sx8_paged.h"

namespace sx8 {
namespace {

constexpr int kPageThreads = 1024;

struct PageTab {
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    int32_t* status;
    int n_slots, max_pages, n_pages, page_tokens;
};

// Workspace: header (count of page pairs, -1: nothing to do), then lists.
struct PageWs {
    int32_t* head;                 // [4]
    int32_t* pages;                // [n_pages] page numbers found
    int32_t* to;                   // [n_pages] compact: where a page went; fork and reserve: first new page by entry
    int32_t* from;                 // [n_pages]
};
int64_t page_ws_bytes(int64_t n_slots, int64_t n_pages) {
    return 16 + 4 * (2 * ((n_pages + 3) / 4 * 4) + ((n_pages > n_slots ? n_pages : n_slots) + 3) / 4 * 4);
}
PageWs page_ws(void* w, int64_t n_pages) {
    int32_t* b = reinterpret_cast<int32_t*>(w);
    const int64_t n4 = (n_pages + 3) / 4 * 4;
    return PageWs{b, b + 4, b + 4 + 2 * n4, b + 4 + n4};
}

// Sum before this thread's v, and the sum of all (one work-group of kPageThreads).
__device__ __forceinline__ int scan_before(int v, int* all) {
    __shared__ int wsum[kPageThreads / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o, 64);
        if (lane >= o) s += u;
    }
    __syncthreads();               // wsum is free again
    if (lane == 63) wsum[w] = s;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kPageThreads / 64; ++i) {
        if (i < w) before += wsum[i];
        sum += wsum[i];
    }
    *all = sum;
    return before + s - v;
}

// The `want` lowest free pages into list (in order); false if there are fewer.  A thread looks at four pages a
// round, so the rounds until enough are found are few.
__device__ __forceinline__ bool find_free(const int32_t* refs, int n_pages, int want, int32_t* list) {
    int have = 0;
    for (int64_t base = 0; base < n_pages && have < want; base += 4 * kPageThreads) {
        const int64_t i0 = base + 4 * (int64_t)threadIdx.x;
        int f[4], n = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = i0 + e < n_pages && refs[i0 + e] == 0;
            n += f[e];
        }
        int all, at = have + scan_before(n, &all);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f[e]) {
                if (at < want) list[at] = (int32_t)(i0 + e);
                ++at;
            }
        have += all;
    }
    __syncthreads();               // the list is written (by this work-group, which reads it)
    return have >= want;
}

// The smallest failing (code, item) of the work-group's threads: code 0 = none.
__device__ __forceinline__ int worst(int code, int item, int* which) {
    __shared__ unsigned long long best;
    if (threadIdx.x == 0) best = ~0ull;
    __syncthreads();
    if (code) atomicMin(&best, (unsigned long long)(unsigned)item << 32 | (unsigned)code);
    __syncthreads();
    const unsigned long long b = best;
    *which = b == ~0ull ? 0 : (int)(b >> 32);
    return b == ~0ull ? 0 : (int)(b & 0xFFFFFFFFu);
}
__device__ __forceinline__ void report(int32_t* status, int code, int item) {
    if (threadIdx.x == 0 && status[0] == 0) {
        status[0] = code;
        status[1] = item;
    }
}

// ---- reserve -----------------------------------------------------------------------------------
__device__ __forceinline__ void clear_mark(int32_t* of) {
    if (*of == kMarkAll) return;                                     // (no bit is set)
#pragma unroll
    for (int i = 0; i < kMarkWords; ++i) of[i] = i ? 0 : kMarkAll;
}

__global__ __launch_bounds__(kPageThreads) void k_reserve(const PageTab t, const int32_t* add, const PageWs ws, int32_t* marks) {
    const int tid = threadIdx.x, pt = t.page_tokens;
    const int64_t cap = (int64_t)t.max_pages * pt;
    int total = 0, code = 0, item = 0;
    for (int s0 = 0; s0 < t.n_slots; s0 += kPageThreads) {
        const int s = s0 + tid;
        int need = 0;
        if (s < t.n_slots) {
            const int64_t len = t.lens[s], a = add[s];
            const int bad = a < 0 || len < 0 || len > cap ? 1 : len + a > cap ? 3 : 0;
            if (bad && !code) {
                code = bad;
                item = s;
            }
            if (!bad) need = (int)((len + a + pt - 1) / pt - (len + pt - 1) / pt);
        }
        int all;
        const int before = total + scan_before(need, &all);
        if (s < t.n_slots) ws.to[s] = before;
        total = total + all < 0 || total + all > t.n_pages ? t.n_pages + 1 : total + all;   // (too many is too many)
    }
    code = worst(code, item, &item);
    if (!code && (total > t.n_pages || !find_free(t.refs, t.n_pages, total, ws.pages))) {
        code = 2;
        item = 0;
    }
    if (code) {
        report(t.status, code, item);
        if (marks)
            for (int s = tid; s < t.n_slots; s += kPageThreads)
                if (add[s] != 0) marks[kMarkWords * s] = kMarkRefused;
        return;
    }
    for (int s = tid; s < t.n_slots; s += kPageThreads) {
        const int len = t.lens[s], a = add[s];
        const int have = (int)(((int64_t)len + pt - 1) / pt), end = (int)(((int64_t)len + a + pt - 1) / pt);
        int at = ws.to[s];
        for (int i = have; i < end; ++i, ++at) {
            const int page = ws.pages[at];
            t.table[(int64_t)s * t.max_pages + i] = page;
            t.refs[page] = 1;
        }
        if (a) {
            t.lens[s] = len + a;
            if (marks) clear_mark(marks + kMarkWords * s);
        }
    }
}

// ---- fork --------------------------------------------------------------------------------------
__global__ __launch_bounds__(kPageThreads) void k_fork(const PageTab t, const int32_t* src, const int32_t* dst, int n,
                                                       const PageWs ws) {
    __shared__ uint32_t is_dst[kKv4MaxSlots / 32], is_src[kKv4MaxSlots / 32];
    const int tid = threadIdx.x, pt = t.page_tokens;
    const int64_t cap = (int64_t)t.max_pages * pt;
    for (int i = tid; i < kKv4MaxSlots / 32; i += kPageThreads) is_dst[i] = is_src[i] = 0;
    __syncthreads();
    int total = 0, code = 0, item = 0;
    auto flag = [&](int c, int i) {
        if (!code) {
            code = c;
            item = i;
        }
    };
    for (int i0 = 0; i0 < n; i0 += kPageThreads) {
        const int i = i0 + tid;
        int need = 0;
        if (i < n) {
            const int a = src[i], b = dst[i];
            if (a < 0 || a >= t.n_slots || b < 0 || b >= t.n_slots || t.lens[a] < 0 || t.lens[a] > cap) {
                flag(1, i);
            } else {
                if (t.lens[b] != 0) flag(4, i);
                // (named twice: no entry is reported, since which of the two comes second is up to the threads)
                if (atomicOr(&is_dst[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) flag(4, 0x7FFFFFFF);
                atomicOr(&is_src[a >> 5], 1u << (a & 31));
                need = t.lens[a] % pt != 0;
            }
        }
        int all;
        const int before = total + scan_before(need, &all);
        if (i < n) ws.to[i] = need ? before : -1;
        total += all;
    }
    __syncthreads();
    for (int i = tid; i < kKv4MaxSlots / 32; i += kPageThreads)
        if (is_dst[i] & is_src[i]) flag(4, 0x7FFFFFFF);
    code = worst(code, item, &item);
    if (!code && !find_free(t.refs, t.n_pages, total, ws.pages)) {
        code = 2;
        item = 0;
    }
    if (tid == 0) ws.head[0] = code ? -1 : n;
    if (code) {
        report(t.status, code, item == 0x7FFFFFFF ? 0 : item);
        return;
    }
    for (int i = tid; i < n; i += kPageThreads) {
        const int a = src[i], b = dst[i], len = t.lens[a], at = ws.to[i];
        t.lens[b] = len;
        if (at >= 0) {
            const int page = ws.pages[at];
            t.table[(int64_t)b * t.max_pages + len / pt] = page;
            t.refs[page] = 1;
            ws.from[at] = t.table[(int64_t)a * t.max_pages + len / pt];
        }
    }
}

constexpr int kChunk = 4096 * 4;           // bytes that a work-group moves between two looks at its list

// 16 bytes a thread, four requested together; chunk c of a page
__device__ __forceinline__ void copy_chunk(uint8_t* dst, const uint8_t* src, int64_t c, int64_t page_bytes) {
    const int64_t base = c * kChunk + 16 * threadIdx.x;
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (base + 4096 * i < page_bytes) v[i] = *reinterpret_cast<const u32x4*>(src + base + 4096 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (base + 4096 * i < page_bytes) *reinterpret_cast<u32x4*>(dst + base + 4096 * i) = v[i];
}

// grid (entries, chunks of a page x layers): the pages' bytes, and (y = 0) the rest of the entry's table row.
__global__ __launch_bounds__(256) void k_fork_copy(uint8_t* pages, int64_t page_bytes, int chunks, const PageTab t,
                                                   const int32_t* src, const int32_t* dst, const PageWs ws) {
    if (ws.head[0] < 0) return;
    const int i = blockIdx.x, a = src[i], b = dst[i], at = ws.to[i];
    const int full = t.lens[a] / t.page_tokens;
    if (blockIdx.y == 0) {
        const int32_t* ra = t.table + (int64_t)a * t.max_pages;
        int32_t* rb = t.table + (int64_t)b * t.max_pages;
        for (int j = threadIdx.x; j < t.max_pages; j += 256) {
            if (j < full) {
                const int page = ra[j];
                rb[j] = page;
                if (page >= 0 && page < t.n_pages) atomicAdd(&t.refs[page], 1);
            } else if (j > full || at < 0) {
                rb[j] = -1;
            }
        }
    }
    if (at < 0) return;
    const int from = ws.from[at], to = ws.pages[at];
    if (from < 0 || from >= t.n_pages) return;
    const int64_t layer = (int64_t)(blockIdx.y / chunks) * t.n_pages * page_bytes;
    copy_chunk(pages + layer + to * page_bytes, pages + layer + from * page_bytes, blockIdx.y % chunks, page_bytes);
}

// ---- free --------------------------------------------------------------------------------------
// Work-group i takes entry i, unless an earlier entry names the same slot.  Every work-group looks at all entries, so all
// of them decide alike whether the call is a valid one.
__global__ __launch_bounds__(256) void k_free(const PageTab t, const int32_t* slots, int n) {
    const int i = blockIdx.x, mine = slots[i];
    int bad = n, twice = 0;
    for (int j = threadIdx.x; j < n; j += 256) {
        const int s = slots[j];
        if (s < 0 || s >= t.n_slots) bad = bad < j ? bad : j;
        if (j < i && s == mine) twice = 1;
    }
    twice = __syncthreads_or(twice);
    if (__syncthreads_or(bad < n)) {
        if (i == 0) {
            int item;
            const int code = worst(bad < n, bad, &item);
            report(t.status, code, item);
        }
        return;
    }
    if (twice) return;
    for (int j = threadIdx.x; j < t.max_pages; j += 256) {
        const int page = t.table[(int64_t)mine * t.max_pages + j];
        if (page >= 0 && page < t.n_pages) atomicSub(&t.refs[page], 1);
        t.table[(int64_t)mine * t.max_pages + j] = -1;
    }
    if (threadIdx.x == 0) t.lens[mine] = 0;
}

// ---- compact -----------------------------------------------------------------------------------
__global__ __launch_bounds__(kPageThreads) void k_compact(const PageTab t, const PageWs ws) {
    const int n = t.n_pages;
    int used = 0;
    for (int64_t i = 4 * (int64_t)threadIdx.x; i < n; i += 4 * kPageThreads)
#pragma unroll
        for (int e = 0; e < 4; ++e) used += i + e < n && t.refs[i + e] != 0;
    int count;
    scan_before(used, &count);
    // free places below count into pages, used pages at or above it into from, in order: as many of one as of the other
    int holes = 0, movers = 0;
    for (int64_t base = 0; base < n; base += 4 * kPageThreads) {
        const int64_t i0 = base + 4 * (int64_t)threadIdx.x;
        int hole[4], mover[4], nh = 0, nm = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = i0 + e < n, u = in && t.refs[i0 + e] != 0;
            hole[e] = in && i0 + e < count && !u;
            mover[e] = u && i0 + e >= count;
            nh += hole[e];
            nm += mover[e];
        }
        // (both counts in one scan: at most 4096 each a round)
        int all;
        const int at = scan_before(nh | nm << 16, &all);
        int ah = holes + (at & 0xFFFF), am = movers + (at >> 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (hole[e]) ws.pages[ah++] = (int32_t)(i0 + e);
            if (mover[e]) ws.from[am++] = (int32_t)(i0 + e);
        }
        holes += all & 0xFFFF;
        movers += all >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < holes; i += kPageThreads) {
        const int to = ws.pages[i], from = ws.from[i];
        ws.to[from] = to;
        t.refs[to] = t.refs[from];
        t.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        ws.head[0] = holes;
        ws.head[1] = count;
    }
}

// Every work-group: its part of the tables, then chunks of the moved pages of every layer in turn.  Source pages lie at or
// above the count and target pages below it, so no copy reads what another writes.
__global__ __launch_bounds__(256) void k_compact_copy(uint8_t* pages, int64_t page_bytes, int chunks, int64_t n_layers,
                                                      const PageTab t, const PageWs ws) {
    const int moved = ws.head[0], count = ws.head[1];
    if (moved == 0) return;
    const int64_t entries = (int64_t)t.n_slots * t.max_pages, stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += stride) {
        const int page = t.table[i];
        if (page >= count && page < t.n_pages) t.table[i] = ws.to[page];
    }
    const int64_t tasks = moved * n_layers * chunks;
    for (int64_t k = blockIdx.x; k < tasks; k += gridDim.x) {
        const int64_t c = k % chunks, r = k / chunks, i = r % moved, layer = r / moved * t.n_pages * page_bytes;
        copy_chunk(pages + layer + ws.pages[i] * page_bytes, pages + layer + ws.from[i] * page_bytes, c, page_bytes);
    }
}

// ---- keep --------------------------------------------------------------------------------------
// Workspace of keep: header (0: nothing to do), then by slot the tokens before its new rows and where its pages begin
// in a list of those pages, which the table loses before the rows move.
struct KeepWs {
    int32_t* head;                 // [4]
    int32_t* base;                 // [n_slots]
    int32_t* at;                   // [n_slots]
    int32_t* pages;                // [rows / page_tokens + 2 n_slots]
};
int64_t keep_ws_bytes(int64_t n_slots, int64_t rows) { return 16 + 4 * (2 * n_slots + rows / 32 + 2 * n_slots); }
KeepWs keep_ws(void* w, int64_t n_slots) {
    int32_t* b = reinterpret_cast<int32_t*>(w);
    return KeepWs{b, b + 4, b + 4 + n_slots, b + 4 + 2 * n_slots};
}

// A slot of n new rows keeps rows path[0] < path[1] < .. (counts of them) of these.  A slot that its reservation was refused
// has none (its last n tokens are older ones): it is passed over.
__global__ __launch_bounds__(kPageThreads) void k_keep(const PageTab t, const int32_t* path, const int32_t* counts,
                                                       const int32_t* cu, Kv4Shape sh, const KeepWs ws, int32_t* marks) {
    const int tid = threadIdx.x, pt = t.page_tokens;
    const int64_t cap = (int64_t)t.max_pages * pt;
    int code = 0, item = 0, total = 0;
    for (int s0 = 0; s0 < t.n_slots; s0 += kPageThreads) {
        const int s = s0 + tid;
        int held = 0;                                                // pages with new rows
        if (s < t.n_slots) {
            int first, n;
            kv4_rows(sh, cu, s, &first, &n);
            const int len = t.lens[s], c = counts[s], base = len - n;
            const int32_t* const of = marks + kMarkWords * s;
            const int mark = n > 0 && marks ? *of : kMarkAll;
            bool bad = false, missing = false;
            if (mark < 0) {
                n = 0;
            } else if (n > 0) {
                bad = c < 0 || c > n || base < 0 || len > cap;
                for (int i = 0, last = -1; !bad && i < c; i += 8) {  // (eight asked for together)
                    int at[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) at[u] = path[first + min(i + u, c - 1)];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        if (i + u >= c) continue;
                        bad |= at[u] <= last || at[u] >= n;
                        last = at[u];
                    }
                }
                for (int i = 0; !bad && mark != kMarkAll && i < c; ++i) {
                    const int r = path[first + i];
                    missing |= r < kMarkRows ? of[1 + r / 32] >> r % 32 & 1 : r >= mark;
                }
                if (!bad) held = (len + pt - 1) / pt - base / pt;
            } else {
                bad = c != 0;
            }
            if ((bad || missing) && !code) {
                code = bad ? 1 : 5;
                item = s;
            }
            ws.base[s] = n > 0 ? base : -1;
        }
        int all;
        const int before = total + scan_before(held, &all);
        if (s < t.n_slots) ws.at[s] = before;
        total = total + all < 0 ? 0x7FFFFFFF : total + all;
    }
    // (a cu that runs backwards can name more rows than there are)
    if (!code && total > sh.rows / 32 + 2 * t.n_slots) {
        code = 1;
        item = 0;
    }
    code = worst(code, item, &item);
    if (tid == 0) ws.head[0] = code == 0;
    if (code) {
        report(t.status, code, item);
        return;
    }
    for (int s = tid; s < t.n_slots; s += kPageThreads) {
        const int base = ws.base[s], len = t.lens[s], at = ws.at[s];
        if (base < 0) continue;
        const int end = base + counts[s], have = (end + pt - 1) / pt;
        for (int i = base / pt; i < (len + pt - 1) / pt; ++i) {
            const int64_t e = (int64_t)s * t.max_pages + i;
            const int page = t.table[e];
            ws.pages[at + i - base / pt] = page;
            if (i >= have) {
                if (page >= 0 && page < t.n_pages) atomicSub(&t.refs[page], 1);
                t.table[e] = -1;
            }
        }
        t.lens[s] = end;
        if (marks) clear_mark(marks + kMarkWords * s);
    }
}

// Work-group (slot, head, layer): the kept rows, a block of the places they go to at a time.  Rows only move to
// the front, so a block's rows come from it or from later ones: read all of them, then write.  K's words belong to one
// token each; a V word holds eight tokens of a dimension and keeps those that are not replaced.
template <int HD>
__global__ __launch_bounds__(256) void k_keep_move(uint8_t* pages, const int32_t* path, const int32_t* counts,
                                                   const int32_t* cu, Kv4Shape sh, int page_tokens, int64_t n_pages,
                                                   int64_t page_bytes, const KeepWs ws) {
    constexpr int kBB = kv4_block_bytes(HD), NG = HD / kKv4Group, kK = 32 * (HD / 8) / 256, kV = 4 * HD / 256 > 0 ? 4 * HD / 256 : 1;
    constexpr int kP = (32 * 4 * NG + 255) / 256;
    __shared__ const uint8_t* from[32];                              // block of the row that goes to token t, null: none
    __shared__ int row[32];                                          // and its token there
    const int s = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    int first, n;
    kv4_rows(sh, cu, s, &first, &n);
    if (n == 0 || ws.head[0] == 0 || ws.base[s] < 0) return;
    const int c = counts[s];
    if (c == 0 || path[first + c - 1] == c - 1) return;              // (they lie together already)
    const int base = ws.base[s], bpp = page_tokens / 32;
    const int32_t* const list = ws.pages + ws.at[s];
    uint8_t* const layer = pages + (int64_t)blockIdx.z * n_pages * page_bytes + (int64_t)head * bpp * kBB;
    auto block = [&](int pos) -> uint8_t* {
        const int page = list[pos / page_tokens - base / page_tokens];
        return page < 0 || page >= n_pages ? nullptr : layer + page * page_bytes + (int64_t)(pos % page_tokens / 32) * kBB;
    };
    for (int b = base / 32; b * 32 < base + c; ++b) {
        uint8_t* const dst = block(b * 32 < base ? base : b * 32);
        __syncthreads();                                             // (the list of the last block is read)
        // (every wave finds them; the first one writes them down)
        const int lane = tid & 63, i = b * 32 + lane - base;
        const uint8_t* src = nullptr;
        if (lane < 32 && i >= 0 && i < c) {
            const int at = path[first + i];
            if (at != i) src = block(base + at);
            if (tid < 32) row[lane] = (base + at) % 32;
        }
        if (tid < 32) from[lane] = src;
        const uint32_t moves = (uint32_t)__builtin_amdgcn_ballot_w64(src != nullptr);
        __syncthreads();
        if (moves == 0 || dst == nullptr) continue;
        uint32_t k[kK], v[kV];
        uint16_t prm[kP];
#pragma unroll
        for (int u = 0; u < kK; ++u) {
            const int i = tid + 256 * u, t = i % 32, d = i / 32 * 8;
            if (moves >> t & 1u) k[u] = *reinterpret_cast<const uint32_t*>(from[t] + kv4_k_word(HD, row[t], d));
        }
#pragma unroll
        for (int u = 0; u < kV; ++u) {
            const int i = tid + 256 * u, d = i % HD, h = __builtin_amdgcn_readfirstlane(i / HD);   // (HD >= 64: a wave's alike)
            if (i >= 4 * HD || !(moves >> 4 * h & 0x000F000Fu)) continue;
            v[u] = *reinterpret_cast<const uint32_t*>(dst + kv4_v_word(HD, 4 * h, d));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = e / 4 * 16 + 4 * h + e % 4;
                if (!(moves >> t & 1u)) continue;
                const uint32_t lv = *reinterpret_cast<const uint32_t*>(from[t] + kv4_v_word(HD, row[t], d)) >> kv4_v_shift(row[t]) & 15u;
                v[u] = (v[u] & ~(15u << kv4_shift(e))) | lv << kv4_shift(e);
            }
        }
#pragma unroll
        for (int u = 0; u < kP; ++u) {
            const int i = tid + 256 * u, t = i % 32, which = i / 32 % 4, g = i / 128;
            if (g < NG && moves >> t & 1u) prm[u] = *reinterpret_cast<const uint16_t*>(from[t] + kv4_param(HD, which, row[t], g));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kK; ++u) {
            const int i = tid + 256 * u, t = i % 32, d = i / 32 * 8;
            if (moves >> t & 1u) *reinterpret_cast<uint32_t*>(dst + kv4_k_word(HD, t, d)) = k[u];
        }
#pragma unroll
        for (int u = 0; u < kV; ++u) {
            const int i = tid + 256 * u, d = i % HD, h = __builtin_amdgcn_readfirstlane(i / HD);
            if (i < 4 * HD && moves >> 4 * h & 0x000F000Fu) *reinterpret_cast<uint32_t*>(dst + kv4_v_word(HD, 4 * h, d)) = v[u];
        }
#pragma unroll
        for (int u = 0; u < kP; ++u) {
            const int i = tid + 256 * u, t = i % 32, which = i / 32 % 4, g = i / 128;
            if (g < NG && moves >> t & 1u) *reinterpret_cast<uint16_t*>(dst + kv4_param(HD, which, t, g)) = prm[u];
        }
    }
}

int32_t make_tab(const char* what, PageTab* t, int32_t* table, int32_t* lens, int32_t* refs, int64_t n_slots,
                 int64_t max_pages, int64_t n_pages, int32_t page_tokens, int32_t* status) {
    if (!table || !refs) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    if (page_tokens != 32 && page_tokens != 64 && page_tokens != 128 && page_tokens != 256)
        return fail(SX8_ERR_INVALID, "%s: page_tokens must be 32, 64, 128 or 256", what);
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || max_pages <= 0 || max_pages * page_tokens > kKv4MaxTokens ||
        n_pages <= 0 || n_pages > 1 << 28)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_slots 1..%d, max_pages * page_tokens 1..%lld, n_pages 1..2^28)", what,
                    kKv4MaxSlots, (long long)kKv4MaxTokens);
    if (!aligned(table, 4) || !aligned(lens, 4) || !aligned(refs, 4) || !aligned(status, 4))
        return fail(SX8_ERR_INVALID, "%s: table, lens, refs and status must be 4-byte aligned", what);
    *t = PageTab{table, lens, refs, status, (int)n_slots, (int)max_pages, (int)n_pages, page_tokens};
    return SX8_OK;
}
int32_t check_ws(const char* what, const void* ws, int64_t bytes, int64_t n_slots, int64_t n_pages) {
    if (!ws || bytes < page_ws_bytes(n_slots, n_pages) || !aligned(ws, 16))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 16-byte aligned", what,
                    (long long)page_ws_bytes(n_slots, n_pages));
    return SX8_OK;
}
int32_t check_pages(const char* what, const uint8_t* pages, int64_t n_layers, int64_t page_bytes) {
    if (!pages || !aligned(pages, 16)) return fail(SX8_ERR_INVALID, "%s: pages must be a 16-byte aligned pointer", what);
    if (n_layers <= 0 || n_layers > 4096 || page_bytes <= 0 || page_bytes % 16 || page_bytes > (int64_t)1 << 30)
        return fail(SX8_ERR_INVALID, "%s: bad sizes (n_layers 1..4096, page_bytes a multiple of 16 up to 2^30)", what);
    return SX8_OK;
}

}  // namespace
}  // namespace sx8

extern "C" int64_t sx8_kv4_pages_workspace_bytes(int64_t n_slots, int64_t n_pages) {
    using namespace sx8;
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || n_pages <= 0 || n_pages > 1 << 28) return -1;
    return page_ws_bytes(n_slots, n_pages);
}

extern "C" int32_t sx8_kv4_reserve(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* add, int64_t n_slots,
                                   int64_t max_pages, int64_t n_pages, int32_t page_tokens, int32_t* status,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    return sx8_kv4_reserve_marked(table, lens, refs, add, n_slots, max_pages, n_pages, page_tokens, status, nullptr, workspace,
                                  workspace_bytes, stream);
}

extern "C" int32_t sx8_kv4_reserve_marked(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* add, int64_t n_slots,
                                          int64_t max_pages, int64_t n_pages, int32_t page_tokens, int32_t* status,
                                          int32_t* marks, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_reserve";
    if (!lens || !add || !status) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    PageTab t;
    int32_t rc = make_tab(what, &t, table, lens, refs, n_slots, max_pages, n_pages, page_tokens, status);
    if (rc == SX8_OK) rc = check_ws(what, workspace, workspace_bytes, n_slots, n_pages);
    if (rc != SX8_OK) return rc;
    if (!aligned(marks, 4)) return fail(SX8_ERR_INVALID, "%s: marks must be 4-byte aligned", what);
    hipLaunchKernelGGL(k_reserve, dim3(1), dim3(kPageThreads), 0, as_stream(stream), t, add, page_ws(workspace, n_pages), marks);
    return check_launch(what);
}

extern "C" int32_t sx8_kv4_fork(uint8_t* pages, int64_t n_layers, int64_t page_bytes, int32_t* table, int32_t* lens,
                                int32_t* refs, const int32_t* src, const int32_t* dst, int64_t n, int64_t n_slots,
                                int64_t max_pages, int64_t n_pages, int32_t page_tokens, int32_t* status,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_fork";
    if (!lens || !status || (n != 0 && (!src || !dst))) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    PageTab t;
    int32_t rc = make_tab(what, &t, table, lens, refs, n_slots, max_pages, n_pages, page_tokens, status);
    if (rc == SX8_OK) rc = check_ws(what, workspace, workspace_bytes, n_slots, n_pages);
    if (rc == SX8_OK) rc = check_pages(what, pages, n_layers, page_bytes);
    if (rc != SX8_OK) return rc;
    if (n < 0 || n > n_slots) return fail(SX8_ERR_INVALID, "%s: n must be 0..n_slots", what);
    const int64_t chunks = (page_bytes + kChunk - 1) / kChunk;
    if (chunks * n_layers > 65535) return fail(SX8_ERR_UNSUPPORTED, "%s: over 1 GiB a page over the layers", what);
    if (n == 0) return ok();
    const PageWs ws = page_ws(workspace, n_pages);
    hipLaunchKernelGGL(k_fork, dim3(1), dim3(kPageThreads), 0, as_stream(stream), t, src, dst, (int)n, ws);
    hipLaunchKernelGGL(k_fork_copy, dim3((unsigned)n, (unsigned)(chunks * n_layers)), dim3(256), 0, as_stream(stream), pages,
                       page_bytes, (int)chunks, t, src, dst, ws);
    return check_launch(what);
}

extern "C" int32_t sx8_kv4_free(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* slots, int64_t n,
                                int64_t n_slots, int64_t max_pages, int64_t n_pages, int32_t* status, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_free";
    if (!lens || !status || (n != 0 && !slots)) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    PageTab t;
    const int32_t rc = make_tab(what, &t, table, lens, refs, n_slots, max_pages, n_pages, 32, status);
    if (rc != SX8_OK) return rc;
    if (n < 0 || n > kKv4MaxSlots) return fail(SX8_ERR_INVALID, "%s: n must be 0..%d", what, kKv4MaxSlots);
    if (n == 0) return ok();
    hipLaunchKernelGGL(k_free, dim3((unsigned)n), dim3(256), 0, as_stream(stream), t, slots, (int)n);
    return check_launch(what);
}

extern "C" int32_t sx8_kv4_compact(uint8_t* pages, int64_t n_layers, int64_t page_bytes, int32_t* table, int32_t* refs,
                                   int64_t n_slots, int64_t max_pages, int64_t n_pages, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_compact";
    PageTab t;
    int32_t rc = make_tab(what, &t, table, nullptr, refs, n_slots, max_pages, n_pages, 32, nullptr);
    if (rc == SX8_OK) rc = check_ws(what, workspace, workspace_bytes, n_slots, n_pages);
    if (rc == SX8_OK) rc = check_pages(what, pages, n_layers, page_bytes);
    if (rc != SX8_OK) return rc;
    const PageWs ws = page_ws(workspace, n_pages);
    const int64_t chunks = (page_bytes + kChunk - 1) / kChunk;
    // as many work-groups as pages can move (no more than half of the pages do), up to eight a CU
    const int64_t most = (n_pages / 2 + 1) * n_layers * chunks;
    hipLaunchKernelGGL(k_compact, dim3(1), dim3(kPageThreads), 0, as_stream(stream), t, ws);
    hipLaunchKernelGGL(k_compact_copy, dim3((unsigned)(most < 2048 ? most : 2048)), dim3(256), 0, as_stream(stream), pages,
                       page_bytes, (int)chunks, n_layers, t, ws);
    return check_launch(what);
}

extern "C" int64_t sx8_kv4_keep_workspace_bytes(int64_t n_slots, int64_t rows) {
    using namespace sx8;
    if (n_slots <= 0 || n_slots > kKv4MaxSlots || rows < 0 || rows > 0x7FFFFFFF) return -1;
    return keep_ws_bytes(n_slots, rows);
}

extern "C" int32_t sx8_kv4_keep(uint8_t* pages, int64_t n_layers, int32_t* table, int32_t* lens, int32_t* refs,
                                const int32_t* cu, const int32_t* path, const int32_t* counts, int64_t rows, int64_t n_slots,
                                int64_t max_pages, int64_t n_pages, int32_t nk, int32_t hd, int32_t page_tokens,
                                int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
    return sx8_kv4_keep_marked(pages, n_layers, table, lens, refs, cu, path, counts, rows, n_slots, max_pages, n_pages, nk, hd,
                               page_tokens, status, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int32_t sx8_kv4_keep_marked(uint8_t* pages, int64_t n_layers, int32_t* table, int32_t* lens, int32_t* refs,
                                       const int32_t* cu, const int32_t* path, const int32_t* counts, int64_t rows,
                                       int64_t n_slots, int64_t max_pages, int64_t n_pages, int32_t nk, int32_t hd,
                                       int32_t page_tokens, int32_t* status, int32_t* marks, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
    using namespace sx8;
    const char* what = "sx8_kv4_keep";
    if (!lens || !status || !counts || (!path && rows > 0)) return fail(SX8_ERR_INVALID, "%s: null pointer", what);
    PageTab t;
    int32_t rc = make_tab(what, &t, table, lens, refs, n_slots, max_pages, n_pages, page_tokens, status);
    if (rc != SX8_OK) return rc;
    const int64_t pb = sx8_kv4_page_bytes(nk, hd, page_tokens);
    if (pb < 0) return fail(SX8_ERR_INVALID, "%s: bad shape (hd 64, 128 or 256, 1 <= nk <= 256)", what);
    rc = check_pages(what, pages, n_layers, pb);
    if (rc != SX8_OK) return rc;
    if (rows < 0 || rows > 0x7FFFFFFF || (!cu && rows != n_slots))
        return fail(SX8_ERR_INVALID, "%s: bad rows (without cu one row a slot)", what);
    if (!aligned(cu, 4) || !aligned(path, 4) || !aligned(counts, 4) || !aligned(marks, 4))
        return fail(SX8_ERR_INVALID, "%s: cu, path, counts and marks must be 4-byte aligned", what);
    if (!workspace || workspace_bytes < keep_ws_bytes(n_slots, rows) || !aligned(workspace, 16))
        return fail(SX8_ERR_INVALID, "%s: workspace needs %lld bytes, 16-byte aligned", what, (long long)keep_ws_bytes(n_slots, rows));
    if (rows == 0) return ok();
    const Kv4Shape sh{(int)n_slots, nk, 1, (int)(max_pages * page_tokens), (int)rows};
    const KeepWs ws = keep_ws(workspace, n_slots);
    hipLaunchKernelGGL(k_keep, dim3(1), dim3(kPageThreads), 0, as_stream(stream), t, path, counts, cu, sh, ws, marks);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)n_slots, (unsigned)nk, (unsigned)n_layers), dim3(256), 0, as_stream(stream),
                           pages, path, counts, cu, sh, page_tokens, n_pages, pb, ws);
    };
    if (hd == 64) go(k_keep_move<64>);
    else if (hd == 128) go(k_keep_move<128>);
    else go(k_keep_move<256>);
    return check_launch(what);
}
