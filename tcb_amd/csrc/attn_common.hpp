// attn_common.hpp -- what the attention kernels over a paged cache share (attn_tokens.hpp, attn_rows.hpp, and attn.hip, which
// plans a call): their arguments, how a batch's rows and keys are cut into work items, the masks, the copies into LDS, and the
// product of one block of keys with a tile of rows.
//
// Rows. The q_heads / kv_heads = G heads that read one kv head are rows of one matrix product: row r of a request's kv
// head h is token r / G, head h G + r % G, so a single token brings G rows and a prompt nq G.
//
// One block: S^T = K Q^T and O^T += V^T P^T on 32x32x16 matrix instructions (fp32 accumulators). In the accumulator of
// S^T lane l holds query l % 32 and the keys 8 g + 4 (l / 32) + r (g, r < 4) in register 4 g + r, so a query's maximum and
// sum are taken over a lane's registers and one exchange between the wave's halves, and rescaling O^T is one multiplier a
// lane. Registers 8 b .. 8 b + 7, rounded to 16 bits, are the second operand of the product over keys 16 b .. 16 b + 15 as
// they stand: its contraction runs over the keys in that register order, and the V^T operand is read in the same order
// (two transposing LDS reads of four keys x sixteen dimensions each). P never leaves its lane.
//
// LDS rows hold their 16-byte chunks in the order chunk ^ swz(row), which spreads both reads (a column of sixteen rows,
// and four rows x 64 bytes) over all banks (measured: no conflict in either); the copies into LDS place a lane's chunk by
// choosing which chunk it fetches.
#pragma once

#include "trhip_internal.hpp"

namespace trhip {

// x / d of 0 <= x < 2^31 for a d of the call's, in a few scalar instructions: floor(x m / 2^(31 + s)), 2^s >= d, m = ceil(2^(31 + s) / d).
// (The excess m d - 2^(31 + s) is below d <= 2^s, so that times x stays below 2^(31 + s).)
struct Div {
    uint32_t m;
    int s;
    void of(int d) {
        s = 0;
        while (((int64_t)1 << s) < d) s++;
        m = (uint32_t)((((uint64_t)1 << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d);
    }
    __device__ __forceinline__ int operator()(int x) const { return (int)(((uint64_t)(uint32_t)x * m) >> (31 + s)); }
};

struct AttnArgs {
    const uint16_t *q;
    uint16_t *out;
    int64_t q_stride, out_stride;  // elements between tokens
    const uint8_t *k, *v;          // cache planes [page][kv head][page rows][dim]
    int64_t page_bytes, npages;
    int head_bytes, page_log2;
    const int *table;
    int64_t max_pages;
    const int *q_start, *kv_len;
    const int *prefix_table;  // shared prefix: pages of its prefix_len keys (0: none)
    int prefix_len, prefix_splits;
    float *prefix_part;  // [split][token][head] partial results of the prefix: DP sums, reference, sum
    int nreq, tokens, heads, kv_heads, group, dim;
    int window, sinks;  // window 0: none
    float scale;        // softmax scale times log2 e
    int out_aligned;    // 8-byte aligned rows
    Div by_group, by_heads;  // by group, kv_heads
    int target, rounds; // workgroups at a time, and how often at most
    int row_lo, row_hi; // requests of row_lo < rows <= row_hi are this launch's
    int part_slots;     // places for the pieces of tiles that are cut (of all tiles behind a prefix), each with an arrival counter
    float *part;        // [place][tile row]: DP sums, then reference (log2 units) and sum of each row
    uint32_t *arrivals;
    int *parts;         // places in use, then for each what the joining launch needs (Place); nullptr: a tile's last workgroup joins it
};

namespace {

typedef __bf16 a8bf __attribute__((ext_vector_type(8)));
typedef _Float16 a8h __attribute__((ext_vector_type(8)));
typedef float a16f __attribute__((ext_vector_type(16)));
typedef short a4s __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uni64(int64_t v) {
    return (int64_t)(((uint64_t)(uint32_t)uni((int)(v >> 32)) << 32) | (uint32_t)uni((int)v));
}
// Wave-uniform int from memory no kernel writes while this one runs: a scalar load (not held up by, and not waiting
// for, the copies into LDS).
__device__ __forceinline__ int sload(const int *p, int64_t i) {
    typedef const __attribute__((address_space(4))) int *cp;
    return ((cp)(uintptr_t)p)[i];
}

template <int DP> __device__ __forceinline__ int swz(int row) {
    return DP == 64 ? 4 * ((row >> 1) & 1) | ((row >> 2) & 3) : 4 * (row & 3) | ((row >> 2) & 3);
}

template <bool BF, class A, class B> __device__ __forceinline__ a16f mma(A a, B b, a16f c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(a8bf, a), __builtin_bit_cast(a8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(a8h, a), __builtin_bit_cast(a8h, b), c, 0, 0, 0);
}

// Two floats rounded to nearest even, packed.
template <bool BF> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, (b2){(__bf16)a, (__bf16)b});
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, (h2){(_Float16)a, (_Float16)b});
    }
}
template <bool BF> __device__ __forceinline__ float wide_lo(uint32_t v) {
    if constexpr (BF) return __uint_as_float(v << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
}
template <bool BF> __device__ __forceinline__ float wide_hi(uint32_t v) {
    if constexpr (BF) return __uint_as_float(v & 0xFFFF0000u);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The same lane of the other half wave: max / sum of both.
__device__ __forceinline__ float half_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));  // (a uint4's members would be read two by two)
__device__ __forceinline__ u32x4 lds16(uint32_t a) {
    typedef const __attribute__((address_space(3))) u32x4 *lp;
    return *(lp)a;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    typedef uint32_t v2 __attribute__((ext_vector_type(2)));
    typedef const __attribute__((address_space(3))) v2 *lp;
    return __builtin_bit_cast(uint2, *(lp)a);
}
__device__ __forceinline__ uint2 lds_tr(uint32_t a) {
    typedef __attribute__((address_space(3))) a4s *lp;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)a));
}

// ---- work items --------------------------------------------------------------------------------------------------------

// The keys a tile of rows reads, in blocks of BK: blocks [0, ns) hold the first tokens that stay visible, blocks
// [w0, w0 + nw) the window (all of the cache without one).
struct Span {
    int ns, w0, nw;
    __device__ __forceinline__ int count() const { return ns + nw; }
    __device__ __forceinline__ int block(int i) const { return i < ns ? i : w0 + (i - ns); }
};
// hi: last visible key of the tile's last token (-1: none), lo: first key of its first token's window
template <int BK> __device__ __forceinline__ Span span_of(int hi, int lo, int sinks) {
    Span s = {0, 0, 0};
    if (hi < 0) return s;
    s.w0 = lo / BK;
    s.nw = hi / BK + 1 - s.w0;
    const int e = sinks < hi + 1 ? sinks : hi + 1;
    s.ns = (e + BK - 1) / BK;
    if (s.ns >= s.w0) {  // no gap: one run from block 0
        s.nw += s.w0;
        s.w0 = 0;
        s.ns = 0;
    }
    return s;
}

// A place's tile, for the launch that joins its pieces: pieces 0: another place has it.
struct Place {
    int pieces, q0, nq, kv, r0, n, head, unused;
};

struct Item {
    int req, tile, split, nsplit, head;
    int q0, nq, kv;  // the request's first token row, new tokens, keys
    int slot;        // its partial result's place (a tile's pieces are kv_heads apart), if it writes one
    int counter;     // place of the tile's piece 0: its arrival counter
    int parts;       // places in use by the launch
};

constexpr int kTokMost = 96;  // rows of a request that goes to attn_tokens (attn.hip)

struct ReqShape {
    int q0, nq, kv, tiles, nb;
};
struct ReqLens {
    int start, end, keys;
};
__device__ __forceinline__ ReqLens lens_of(const AttnArgs &p, int i) {
    ReqLens r = {0, 0, 0};
    if (i < p.nreq) {
        r.start = p.q_start[i];
        r.end = p.q_start[i + 1];
        r.keys = p.kv_len[i];
    }
    return r;
}
template <int TR, int BK> __device__ __forceinline__ ReqShape shape_of(const AttnArgs &p, const ReqLens &r) {
    ReqShape s = {0, 0, 0, 0, 0};
    const int a = r.start < 0 ? 0 : r.start > p.tokens ? p.tokens : r.start, b = r.end < a ? a : r.end > p.tokens ? p.tokens : r.end;
    const int64_t cap = p.max_pages << p.page_log2;
    const int kv = r.keys < 0 ? 0 : (int64_t)r.keys > cap ? (int)cap : r.keys;
    s.q0 = a;
    s.nq = b - a;
    s.kv = kv;
    const int rows = s.nq * p.group;
    if (rows <= p.row_lo || rows > p.row_hi) return s;
    s.tiles = (rows + TR - 1) / TR;
    int keys = kv;
    if (p.window > 0) {
        const int64_t most = (int64_t)p.window + p.sinks + TR + 2 * BK;
        keys = (int64_t)keys > most ? (int)most : keys;
    }
    s.nb = (keys + BK - 1) / BK;
    return s;
}

// How many blocks a piece of a tile's keys has: n tiles of `sum` blocks in all, the longest of `most`, on `target` workgroups
// at a time; starting a piece, writing its result and joining it take as long as `over` blocks. Pieces of at most c
// blocks are at most sum / c + n. Estimated, in blocks, and the least taken:
//   whole tiles       most, where all run at once; else sum / target and half the longest
//   one round         c + over, c = sum / (target - n) (all pieces at once), where n < target
//   dealt out         (sum + over (sum / c + n)) / target + c + over, least at c = sqrt(over sum / target)
// Never more than rounds * target pieces, and none of under `least` blocks.
// Measured, in us, at these constants and at others: kMostRounds 6 (64 tokens of up to 8192 keys 203; 2: 219); kTokLeast 8, two
// blocks a wave (one token x 300 keys 10.6; 4: 10.9, 2: 12.0; x 4096 keys 13.9; 4: 15.1, 16: 15.7; 16 tokens in a window of 256
// 12.3; 4: 14.5; 8 tokens behind 1000 shared keys 13.6; 4: 14.3, 16: 15.2); kTokOver 6 (64 requests of up to 12 tokens 72.6; 3: 78.0;
// 12: the same); kRowsOver 20 (6 prompts of up to 300 tokens 30.1; 10: 34.4); kRowsLeast 6
// (32 tokens behind 4096 shared keys 21.8; 4: 22.7, 2: 27.0).
constexpr int kMostRounds = 6;
constexpr int kRowsLeast = 6, kRowsOver = 20;  // attn_rows: blocks of a piece at least, and what one costs beside them
__host__ __device__ inline int piece_blocks(float sum, int n, int most, int target, int rounds, int least, int over) {
    constexpr int kWhole = 0x40000000;
    // (in floats, made a little larger than they can have been rounded down)
#if defined(__HIP_DEVICE_COMPILE__)
    auto ratio = [](float a, float b) { return a * __builtin_amdgcn_rcpf(b); };
    auto root = [](float a) { return __builtin_amdgcn_sqrtf(a); };
#else
    auto ratio = [](float a, float b) { return a / b; };
    auto root = [](float a) { return sqrtf(a); };
#endif
    const float s = sum * 1.0001f, each = ratio(s, (float)target);
    float best = n <= target ? (float)most : each + 0.5f * (float)most, piece = (float)kWhole;
    if (rounds > 0 && n < target) {
        const float c = fmaxf(ceilf(ratio(s, (float)(target - n))), (float)least);
        if (c + (float)over < best) {
            best = c + (float)over;
            piece = c;
        }
    }
    const int64_t room = (int64_t)rounds * target - n;
    if (room > 0) {
        const float c = fmaxf(ceilf(fmaxf(root((float)over * each), ratio(s, (float)room))), (float)least);
        const float e = each + ratio((float)over * (ratio(s, c) + (float)n), (float)target) + c + (float)over;
        if (e < best) piece = c;
    }
    return piece >= (float)most ? kWhole : (int)piece;
}

// Inclusive sums (or maxima) over the wave's lanes in six lane moves.
template <int CTRL, int ROWS, class T> __device__ __forceinline__ T lane_move(T v, T zero) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, zero), __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
}
template <class T, class F> __device__ __forceinline__ T scan64(T v, T zero, F f) {
    v = f(v, lane_move<0x111, 0xF>(v, zero));  // row_shr 1, 2, 4, 8: within sixteen lanes
    v = f(v, lane_move<0x112, 0xF>(v, zero));
    v = f(v, lane_move<0x114, 0xF>(v, zero));
    v = f(v, lane_move<0x118, 0xF>(v, zero));
    v = f(v, lane_move<0x142, 0xA>(v, zero));  // row_bcast 15, 31: across them
    v = f(v, lane_move<0x143, 0xC>(v, zero));
    return v;
}

struct Plus {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
    __device__ __forceinline__ int operator()(int a, int b) const { return __builtin_elementwise_add_sat(a, b); }  // (starts out of order)
};

// ceil(nb / piece); a batch has few thousand pieces at most (piece_blocks), so a quotient in floats is one off at most.
__device__ __forceinline__ int pieces_of(int nb, int piece) {
    const int x = nb + piece - 1;
    int q = (int)((float)x * __builtin_amdgcn_rcpf((float)piece));
    const int r = x - q * piece;
    q = r < 0 ? q - 1 : r >= piece ? q + 1 : q;
    return nb <= piece ? 1 : q;
}

// Which tile of rows and which piece of its keys workgroup wg takes; every wave finds out for itself (no barrier). A request's
// tiles are all cut into the same number of pieces (piece_blocks). Items are numbered head fastest, then piece, tile (the last
// tokens of a prompt, whose rows read most keys, first), request. False: no item left.
template <int TR, int BK, int CMIN, int OVER> __device__ __forceinline__ bool find_item(const AttnArgs &p, int wg, int grid, Item &it) {
    it = Item{0, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0};
    const int lane = threadIdx.x & 63, x = p.by_heads(wg);
    // The lengths of the first 64 READ requests are read at once (each 64 by themselves are a memory latency more: 128 requests
    // of 1000 keys took 60.5 us so, 58.6 now) and go round in registers, so that the loops stay short: a launch fetches
    // their instructions anew.
    constexpr int READ = 4;
    ReqLens lens[READ] = {};
    lens[0] = lens_of(p, lane);
    if (p.nreq > 64) {
#pragma unroll
        for (int c = 1; c < READ; c++) lens[c] = lens_of(p, 64 * c + lane);
    }
    auto each = [&](auto use) {
        ReqLens at[READ] = {lens[0], lens[1], lens[2], lens[3]};
#pragma unroll 1
        for (int base = 0; base < p.nreq; base += 64) {
            if (base >= 64 * READ) at[0] = lens_of(p, base + lane);
            use(shape_of<TR, BK>(p, at[0]), base);
            at[0] = at[1], at[1] = at[2], at[2] = at[3];
        }
    };
    float sum = 0.0f;
    int tiles = 0, most = 0;
    each([&](const ReqShape &t, int) {
        sum += (float)t.tiles * (float)t.nb;
        tiles = Plus()(tiles, t.tiles);
        most = t.nb > most ? t.nb : most;
    });
    sum = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scan64(sum, 0.0f, Plus())), 63));
    tiles = __builtin_amdgcn_readlane(scan64(tiles, 0, Plus()), 63);
    most = __builtin_amdgcn_readlane(scan64(most, 0, [](int a, int b) { return a > b ? a : b; }), 63);
    const int piece = piece_blocks(sum * (float)p.kv_heads, tiles * p.kv_heads, most, p.target, p.rounds, CMIN, OVER);
    int before = 0, parts = 0;
    bool found = false;
    each([&](const ReqShape &s, int base) {
        const int ns = pieces_of(s.nb, piece), n = s.tiles * ns, np = ns > 1 || p.prefix_splits > 0 ? n : 0;
        const int incl = scan64(n, 0, Plus()), inclp = scan64(np, 0, Plus());
        if (!found) {
            const uint64_t m = __ballot(Plus()(before, incl) > x);
            if (m) {
                const int src = __builtin_ctzll(m);
                it.req = base + src;
                it.q0 = __builtin_amdgcn_readlane(s.q0, src);
                it.nq = __builtin_amdgcn_readlane(s.nq, src);
                it.kv = __builtin_amdgcn_readlane(s.kv, src);
                it.nsplit = __builtin_amdgcn_readlane(ns, src);
                const int start = before + __builtin_amdgcn_readlane(incl - n, src), at = x - start;
                const int t = it.nsplit == 1 ? at : at / it.nsplit, tiles = __builtin_amdgcn_readlane(s.tiles, src);
                it.split = at - t * it.nsplit;
                it.tile = tiles - 1 - t;
                it.head = wg - x * p.kv_heads;
                it.slot = (parts + __builtin_amdgcn_readlane(inclp - np, src) + at) * p.kv_heads + it.head;
                it.counter = it.slot - it.split * p.kv_heads;
                found = true;
            }
        }
        before = Plus()(before, __builtin_amdgcn_readlane(incl, 63));
        parts = Plus()(parts, __builtin_amdgcn_readlane(inclp, 63));
    });
    it.req = uni(it.req), it.tile = uni(it.tile), it.split = uni(it.split), it.nsplit = uni(it.nsplit), it.head = uni(it.head);
    it.q0 = uni(it.q0), it.nq = uni(it.nq), it.kv = uni(it.kv), it.slot = uni(it.slot), it.counter = uni(it.counter);
    it.parts = uni(parts) * p.kv_heads;
    // starts that are not in order could name more items than there are workgroups: then nothing is done
    const bool fits = (int64_t)before * p.kv_heads <= (int64_t)grid && (int64_t)parts * p.kv_heads <= p.part_slots;
    if (!fits) it.parts = 0;
    return found && fits;
}

// ---- a tile's rows and masks -------------------------------------------------------------------------------------------

// What the rows of a tile (or of a wave's share of one) see. Per lane: the row's last visible key and the first of its
// window; per wave: the extremes over all rows.
struct Rows {
    int hi, lo;                          // this lane's row
    int hi_min, hi_max, lo_min, lo_max;  // over the rows
    int sinks;
};

// Rows r0 .. r0 + n - 1 (n >= 1) of a request with nq new tokens and kv keys; lane's row r0 + lane % 32 (clamped to the last).
__device__ __forceinline__ Rows rows_of(const AttnArgs &p, int r0, int n, int nq, int kv) {
    Rows w;
    const int row = r0 + ((int)(threadIdx.x & 31) < n ? (int)(threadIdx.x & 31) : n - 1);
    const int t0 = p.by_group(r0), t1 = p.by_group(r0 + n - 1), t = p.by_group(row), first = kv - nq;
    auto low = [&](int hi) { return p.window > 0 && hi >= p.window ? hi - p.window + 1 : 0; };
    w.hi = first + t;
    w.lo = low(w.hi);
    w.hi_min = uni(first + t0);
    w.hi_max = uni(first + t1);
    w.lo_min = uni(low(first + t0));
    w.lo_max = uni(low(first + t1));
    w.sinks = p.sinks;
    return w;
}

// Sixteen rows of keys (or values) from token t, t a multiple of 16, for the LDS copies of one wave: the page they lie in, if a
// row sees them, and the descriptors. Rows past hi, pieces that no row of the tile sees (between the first tokens and the
// window) and chunks past dim become zeros, whatever the cache holds there, and so do pages out of range. A piece that
// the window's start or the first tokens' end divides comes whole.
__device__ __forceinline__ int page16(const AttnArgs &p, const int *table, int t, int hi) {
    return t <= hi ? sload(table, t >> p.page_log2) : 0;
}
struct Piece16 {
    dma_rsrc k, v;
};
__device__ __forceinline__ Piece16 piece16(const AttnArgs &p, int page, int head, int t, int hi, int lo, int sinks) {
    Piece16 s;
    int cnt = hi + 1 - t;
    cnt = cnt < 0 ? 0 : cnt > 16 ? 16 : cnt;
    if (sinks <= t && lo >= t + 16) cnt = 0;
    if ((uint32_t)page >= (uint32_t)p.npages) {
        page = 0;
        cnt = 0;
    }
    const int64_t off = uni64((int64_t)page * p.page_bytes + (int64_t)head * p.head_bytes + (int64_t)((t & ((1 << p.page_log2) - 1)) * p.dim * 2));
    const uint32_t bytes = (uint32_t)uni(cnt * p.dim * 2);
    s.k = dma_desc(p.k + off, bytes);
    s.v = dma_desc(p.v + off, bytes);
    return s;
}
// Per-lane byte offsets of instruction i's chunks (16 * DP / 512 instructions a piece).
template <int DP> struct Lanes16 {
    static constexpr int N = DP / 32, CH = DP / 8, RPI = 64 / CH;
    uint32_t voff[N];
    __device__ __forceinline__ void init(int dim) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = lane / CH + i * RPI, c = (lane % CH) ^ swz<DP>(r);
            voff[i] = 8 * c < dim ? (uint32_t)(r * dim * 2 + c * 16) : 0x80000000u;
        }
    }
    __device__ __forceinline__ void copy_one(dma_rsrc d, uint32_t dst, int i) const { dma16(d, dst + i * 1024, voff[i], 0); }
    __device__ __forceinline__ void copy(dma_rsrc d, uint32_t dst) const {
#pragma unroll
        for (int i = 0; i < N; i++) copy_one(d, dst, i);
    }
};

// Q^T operands of this lane's row (element 16 s + 8 (lane / 32) + i in q[s]), zeros past dim. Lanes past the tile's rows
// take its first.
template <int DP> __device__ __forceinline__ void load_q(const AttnArgs &p, uint4 (&q)[DP / 16], int q0, int r0, int n, int head) {
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int row = r0 + (r < n ? r : 0), t = p.by_group(row), g = row - t * p.group;
    const uint16_t *src = p.q + (int64_t)(q0 + t) * p.q_stride + (int64_t)(head * p.group + g) * p.dim + 8 * h;
    auto read = [&](int d) {
        uint4 w;
        __builtin_memcpy(&w, src + d, 16);  // (rows need be aligned to their type only)
        return w;
    };
    if (p.dim == DP) {
#pragma unroll
        for (int s = 0; s < DP / 16; s++) q[s] = read(16 * s);
    } else {
#pragma unroll
        for (int s = 0; s < DP / 16; s++) q[s] = read(16 * s + 8 * h < p.dim ? 16 * s : -8 * h);
#pragma unroll
        for (int s = 0; s < DP / 16; s++) q[s] = 16 * s + 8 * h < p.dim ? q[s] : make_uint4(0, 0, 0, 0);
    }
}

// ---- one block of keys -------------------------------------------------------------------------------------------------

// Weights stand in 16 bits relative to a reference m (log2 units): the row's largest weight is 2^kLift to 2^(kLift + 8). f16 has
// normal numbers down to 2^-14 and nothing below 2^-24, so its weights stand as high as they can; bf16 reaches as far as fp32.
template <bool BF> constexpr int kLift = BF ? 0 : 7;
constexpr float kFar = 1048576.0f;  // scores past 2^20 (log2 units) are made relative to another score first

template <int DP> struct Acc {
    a16f o[DP / 32];
    float m, f, l;  // reference; the score it came from; this lane's share of the sum (its half of the keys)
    float most;     // the highest reference so far
    bool far;
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int i = 0; i < DP / 32; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[i][r] = 0.0f;
        m = f = most = -__builtin_inff();
        l = 0.0f;
        far = false;
    }
};

// S^T of 32 keys at LDS address k. All operands are read before the first product (the compiler would read each right
// before its use, an LDS latency a product).
template <int DP, bool BF> __device__ __forceinline__ a16f scores(uint32_t k, const uint4 (&q)[DP / 16]) {
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const uint32_t a = k + r * (2 * DP) + ((h ^ swz<DP>(r)) << 4);
    u32x4 f[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; i++) f[i] = lds16(a ^ (i << 5));
    __builtin_amdgcn_sched_barrier(0);
    a16f s = {};
#pragma unroll
    for (int i = 0; i < DP / 16; i++) s = mma<BF>(f[i], q[i], s);
    return s;
}

// Scores of keys a row does not see become -Inf. t: the block's first key.
__device__ __forceinline__ void mask(a16f &s, const Rows &w, int t) {
    const int b = t + 4 * ((threadIdx.x >> 5) & 1), dh = w.hi - b, dl = w.lo - b, ds = w.sinks - b;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int e = 8 * (i >> 2) + (i & 3);
        s[i] = e <= dh && (e >= dl || e < ds) ? s[i] : -__builtin_inff();
    }
}
// Whether every row sees all of keys t .. t + n - 1.
__device__ __forceinline__ bool all_see(const Rows &w, int t, int n) {
    return t + n - 1 <= w.hi_min && (t >= w.lo_max || t + n <= w.sinks);
}

// Whether 32 rows of values at LDS address v hold an infinity or a NaN (exponent all ones).
template <int DP, bool BF> __device__ __forceinline__ bool odd_values(uint32_t v) {
    constexpr uint32_t E = BF ? 0x7F807F80u : 0x7C007C00u, U = BF ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
        const u32x4 x = lds16(v + i * 1024 + (threadIdx.x & 63) * 16);
        any |= ((x.x & E) + U) | ((x.y & E) + U) | ((x.z & E) + U) | ((x.w & E) + U);
    }
    return __any((any & 0x80008000u) != 0);
}

// O^T += V^T P^T key by key in fp32, a key's values reaching only the rows that see it: for blocks where some rows see
// a key that others do not and some value is not finite (0 times it would reach every row of the tile).
template <int DP, bool BF>
__device__ __forceinline__ void values_one_by_one(a16f (&o)[DP / 32], const a16f &pr, uint32_t v, int hi, int lo, int sinks, int t) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll 1
    for (int k = 0; k < 32; k++) {
        const int reg = 4 * (k >> 3) + (k & 3);
        float x = pr[0];
#pragma unroll
        for (int i = 1; i < 16; i++) x = reg == i ? pr[i] : x;
        x = __shfl(x, (lane & 31) + 32 * ((k >> 2) & 1));
        const int j = t + k;
        const bool see = j <= hi && (j >= lo || j < sinks);
#pragma unroll
        for (int b = 0; b < DP / 32; b++) {
            __builtin_amdgcn_sched_barrier(0);  // a rare path: few registers rather than many reads in flight
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint2 w = lds8(v + k * (2 * DP) + (((4 * b + g) ^ swz<DP>(k)) << 4) + 8 * h);
                const float e[4] = {wide_lo<BF>(w.x), wide_hi<BF>(w.x), wide_lo<BF>(w.y), wide_hi<BF>(w.y)};
#pragma unroll
                for (int r = 0; r < 4; r++) o[b][4 * g + r] = see ? fmaf(x, e[r], o[b][4 * g + r]) : o[b][4 * g + r];
            }
        }
    }
}

// O^T += V^T P^T of 32 keys at LDS address v, P in 16 bits; TWO: in two terms (what the first rounding drops is the
// second), so that P's rounding does not show beside the output's. EARLY: operands are read before the products, where there
// are registers for them.
template <int DP, bool BF, bool TWO, bool EARLY> __device__ __forceinline__ void values(a16f (&o)[DP / 32], const a16f &pr, uint32_t v) {
    const int lane = threadIdx.x & 63, i = lane & 15, h = lane >> 5;
    const int row = 4 * h + (i >> 2), c = 2 * ((lane >> 4) & 1) + ((i >> 1) & 1);
    const uint32_t a = v + row * (2 * DP) + ((c ^ swz<DP>(row)) << 4) + 8 * (i & 1);
    uint4 f[2][DP / 32];
    auto read = [&](int b) {
#pragma unroll
        for (int d = 0; d < DP / 32; d++) {
            const uint32_t at = (a ^ (d << 6)) + b * 32 * DP;
            const uint2 x = lds_tr(at), y = lds_tr((at ^ 32) + 16 * DP);
            f[b][d] = make_uint4(x.x, x.y, y.x, y.y);
        }
    };
    if (EARLY) {
        read(0);
        if (DP <= 128) read(1);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
        if (!EARLY || (DP > 128 && b == 1)) {
            read(b);
            if (!EARLY) __builtin_amdgcn_sched_barrier(0);
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x = pr[8 * b + 2 * j], y = pr[8 * b + 2 * j + 1];
            hi[j] = pack2<BF>(x, y);
            if (TWO) lo[j] = pack2<BF>(x - wide_lo<BF>(hi[j]), y - wide_hi<BF>(hi[j]));
        }
        const uint4 ph = make_uint4(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
        for (int d = 0; d < DP / 32; d++) o[d] = mma<BF>(f[b][d], ph, o[d]);
        if (TWO) {
#pragma unroll
            for (int d = 0; d < DP / 32; d++) o[d] = mma<BF>(f[b][d], make_uint4(lo[0], lo[1], lo[2], lo[3]), o[d]);
        }
    }
}

// The running softmax's step over 32 scores: scores replaced by exp2(scale s - m), m the row's reference, a whole power of two
// (the score itself where that is far from 0). It is raised to the largest score only where that exceeds the one it came from
// by more than 2^8, and O^T and the sum are then rescaled, exactly: weights of up to 2^8 cost no precision, rescaling every
// time a maximum grows cost a quarter of a token step's instructions. A row that has seen nothing keeps m = -Inf and adds nothing.
// f16: where a block's largest weight is below 2^-7 (one early key outweighs the rest), the smaller ones would lose their last bits
// or vanish. The reference is then lowered to that block, by 2^64 in all at most, and O^T and the sum, which are fp32, are scaled up.
template <int DP, bool BF> __device__ __forceinline__ void softmax_step(Acc<DP> &A, a16f &s, float scale) {
    float x = s[0];
#pragma unroll
    for (int i = 0; i < 16; i++) x = fmaxf(x, s[i]);
    x = half_max(x);
    const float d = (x - A.f) * scale;  // (a difference: a sum rounds to the next score where they are far from 0)
    const bool low = !BF && d < -14.0f && x > -__builtin_inff() && !A.far && A.m > A.most - 64.0f;
    if (__any(d > 8.0f || low)) {
        const bool move = d > 8.0f || low;
        float y = x * scale;
        if (!BF) {
            const float least = A.most - 64.0f + kLift<BF>;
            const bool cut = low && y < least;
            y = cut ? least : y;
            x = cut ? least * __builtin_amdgcn_rcpf(scale) : x;
        }
        const bool far = fabsf(y) > kFar;
        const float r = far ? y : ceilf(y) - kLift<BF>;
        const float a = move ? exp2_hw(far && A.far ? (A.f - x) * scale : A.m - r) : 1.0f;  // from -Inf: 0
        A.l *= a;
#pragma unroll
        for (int d = 0; d < DP / 32; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) A.o[d][i] *= a;
        A.m = move ? r : A.m;
        A.f = move ? x : A.f;
        A.far = move ? far : A.far;
        A.most = fmaxf(A.most, A.m);
    }
    // One fused step an element. Where scores are far the difference is taken first.
    const float neg = A.far || A.m == -__builtin_inff() ? 0.0f : -A.m;
    if (__any(A.far)) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] -= A.far ? A.f : 0.0f;
    }
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        s[i] = exp2_hw(fmaf(s[i], scale, neg));
        l += s[i];
    }
    A.l += l;
}

// ---- results -----------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void agent_store(float *p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 agent_load(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Four finished outputs of row `row` (of the request's kv head) from dimension d; l: the row's sum. A row whose mask
// leaves nothing (hi < 0) is 0; a sum of 0 over visible keys is the formula's 0 / 0. A sum of values that is not finite is NaN: of
// an infinity the products leave either (a weight's second term, or the weight in 16 bits, may be 0 or negative), and which must
// not hang on the batch or the block.
template <bool BF> __device__ __forceinline__ void put4(const AttnArgs &p, int q0, int row, int head, int d, const float (&o)[4], float l, bool sees) {
    if (d >= p.dim) return;
    const int t = p.by_group(row), g = row - t * p.group;
    uint16_t *dst = p.out + (int64_t)(q0 + t) * p.out_stride + (int64_t)(head * p.group + g) * p.dim + d;
    const float inv = 1.0f / l;  // one division, an fp32 rounding more
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = sees ? fmaf(o[i], 0.0f, o[i] * inv) : 0.0f;
    const uint2 w = make_uint2(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]));
    if (p.out_aligned) {
        *reinterpret_cast<uint2 *>(dst) = w;
    } else {
        dst[0] = (uint16_t)w.x;
        dst[1] = (uint16_t)(w.x >> 16);
        dst[2] = (uint16_t)w.y;
        dst[3] = (uint16_t)(w.y >> 16);
    }
}

// A sum over partial results of one row: the largest reference so far (in units of log2), sums relative to it.
struct Join {
    float m, l, o[4];
    __device__ __forceinline__ void init() {
        m = -__builtin_inff();
        l = o[0] = o[1] = o[2] = o[3] = 0.0f;
    }
    __device__ __forceinline__ void add(float pm, float pl, float a, float b, float c, float d) {
        const float n = fmaxf(m, pm);
        const float x = m == n ? 1.0f : exp2_hw(m - n), y = pm == n ? 1.0f : exp2_hw(pm - n);
        l = l * x + pl * y;
        o[0] = o[0] * x + a * y;
        o[1] = o[1] * x + b * y;
        o[2] = o[2] * x + c * y;
        o[3] = o[3] * x + d * y;
        m = n;
    }
};

// The last workgroup of a tile joins its pieces (agent-coherent loads: other workgroups of this launch wrote them). The
// WAVES waves take every WAVES-th piece, eight loads of each in flight, and join their sums in LDS (`room` bytes at `lds`).
template <int DP, int TR, bool BF, int WAVES>
__device__ __forceinline__ void join_tile(const AttnArgs &p, const Item &it, int r0, int n, float *lds, int room) {
    constexpr int ST = DP + 2, AT = 8;
    const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), items = n * (DP / 4);
    const int chunk = room / (WAVES * 6 * 4) / 64 * 64;
    const float *src = p.part + (int64_t)it.counter * TR * ST;
    const int64_t step = (int64_t)p.kv_heads * TR * ST;
    for (int c0 = 0; c0 < items; c0 += chunk) {
        const int cnt = items - c0 < chunk ? items - c0 : chunk;
        for (int i = lane; i < cnt; i += 64) {
            const int idx = c0 + i, r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4;
            Join j;
            j.init();
            const float *x = src + r * ST;
            for (int s0 = w; s0 < it.nsplit; s0 += AT * WAVES) {
                float2 a[AT], b[AT], ml[AT];
#pragma unroll
                for (int u = 0; u < AT; u++) {
                    const float *y = x + (s0 + u * WAVES < it.nsplit ? s0 + u * WAVES : s0) * step;
                    a[u] = agent_load(y + d);
                    b[u] = agent_load(y + d + 2);
                    ml[u] = agent_load(y + DP);
                }
#pragma unroll
                for (int u = 0; u < AT; u++)
                    if (s0 + u * WAVES < it.nsplit) j.add(ml[u].x, ml[u].y, a[u].x, a[u].y, b[u].x, b[u].y);
            }
            float *dst = lds + (w * chunk + i) * 6;
            dst[0] = j.m, dst[1] = j.l;
#pragma unroll
            for (int k = 0; k < 4; k++) dst[2 + k] = j.o[k];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < cnt; i += 64 * WAVES) {
            const int idx = c0 + i, r = idx / (DP / 4), d = (idx - r * (DP / 4)) * 4, row = r0 + r;
            Join j;
            j.init();
#pragma unroll
            for (int u = 0; u < WAVES; u++) {
                const float *x = lds + (u * chunk + i) * 6;
                j.add(x[0], x[1], x[2], x[3], x[4], x[5]);
            }
            put4<BF>(p, it.q0, row, it.head, d, j.o, j.l, it.kv - it.nq + p.by_group(row) >= 0);
        }
        __syncthreads();
    }
}

// For the joining launch: this item's place, and (by workgroup 0) how many there are.
__device__ __forceinline__ void leave_place(const AttnArgs &p, const Item &it, int r0, int n) {
    if (threadIdx.x == 0)
        reinterpret_cast<Place *>(p.parts + 8)[it.slot] = Place{it.split == 0 ? it.nsplit : 0, it.q0, it.nq, it.kv, r0, n, it.head, 0};
}
__device__ __forceinline__ void leave_count(const AttnArgs &p, const Item &it, int wg) {
    if (p.parts && wg == 0 && threadIdx.x == 0) p.parts[0] = it.parts;
}

// Partial results are written: whether this workgroup is the last of its tile's pieces.
__device__ __forceinline__ bool last_piece(const AttnArgs &p, const Item &it, int *flag) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);  // this thread's stores have completed
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(&p.arrivals[it.counter], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                          (uint32_t)(it.nsplit - 1);
        if (last) __hip_atomic_store(&p.arrivals[it.counter], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    return *flag != 0;
}

}  // namespace

// attn_two.hip: two kinds of work in one launch. a: what `kind` says, on na workgroups; b: few rows, on nb.
enum class TwoKind { Rows, PrefixRows, PrefixTokens };
int launch_attn_two(trhip_ctx *ctx, const AttnArgs &a, int na, TwoKind kind, const AttnArgs &b, int nb, int dp, bool bf, int turn);
// attn_rows.hip: rows of a tile and keys of a block, and the launch.
int attn_rows_per_cu(int dp);
int attn_rows_tile();
int attn_rows_block();
int launch_attn_rows(trhip_ctx *ctx, const AttnArgs &p, int dp, bool bf, bool prefix, int64_t grid);
int launch_attn_rows256(trhip_ctx *ctx, const AttnArgs &p, bool bf, bool prefix, int64_t grid);  // attn_rows256.hip

}  // namespace trhip
