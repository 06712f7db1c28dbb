// attn4.hip -- attention over the 4-bit paged cache (kv4.hpp) for few rows, and the call's plan.
//
// Rows, work items, pieces and joins are those of the 16-bit cache's kernel of few rows (attn_common.hpp): a workgroup takes a tile of
// 16 rows (the heads of a few tokens that read one kv head) and a piece of the keys; its four waves take every fourth block of
// 32 keys and join through LDS. What differs is the block. (Tiles of 32 rows open a block's codes once for two products, but hold half as many
// waves a CU: 64 requests of up to 12 tokens, 2000 keys, took 57 us against 43, of up to 24 tokens, 8192 keys, 220 against 186.)
//
// Nothing of a block goes through LDS: the codes lie in memory as the matrix instructions' operands want them, so a lane loads
// its part of a piece of sixteen places as it stands. Two nibbles c masked out of a dword become 1024 + c (or 64 + c) in f16 by
// setting the exponent, and c - 8, exactly, by one packed subtraction: nine instructions open eight codes. (Left as c 2^-24, below f16's
// normal range, five would do, but the matrix units sum such products to 2^-18 only.)
//   S^T of a block of 32 elements: q.(c - 8), then times the key's scale, in fp32, summed over the blocks. q is scaled by a power of two
//   to f16's upper end.
//   O^T += V^T P^T: the value's scale goes to the weight, w = p s (there is one product a block of 32 elements).
// The weights p s stand in f16, in one term for bf16 results (their rounding of 2^-12 is a sixteenth of the result's) and in two
// for f16 ones. (Two for bf16 as well: 64 x 8192 tokens take 82.4 us against 76.7, 64 requests of up to 12 tokens 46.7 against 41; the results' error
// against 64 bits is then 0.001666 of them, which is their own rounding, with one term 0.001679.) So that they neither overflow nor vanish, the softmax's reference includes the largest scale the row has seen.
//
// A wave copies its next block's pieces into LDS while it works on one in registers (loads into registers instead: 64 x 8192 tokens 119 us
// against 97 at that step; copies two blocks ahead 77 against 75, with heads of 64 47 against 43). What bounds it is its instructions beside the bytes: 64 tokens of 32 heads on 8 of 128, up to 8192 keys, bf16: 75 to 81 us
// (3.8 to 4.0 TB/s of codes and scales), vector units busy half the time, matrix units a twelfth. A token over 131071 keys, f16: 45 to 48 us;
// over 300 keys: 8.5, most of it the chain of one block after the other.
#include "attn4_image.hpp"
#include "attn_plan.hpp"
#include "kv4.hpp"

namespace trhip {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// Bytes of a plane of opened keys at most: with both a seventieth of the memory. Where the keys of long requests are opened first, a prompt of
// 8192 tokens takes 525 us, read as they are 1278; 8 prompts of up to 901 beside 32 tokens, window 1000: 87 and 105.
constexpr int64_t kMostImage = (int64_t)2 << 30;
// Calls so small that the two launches more and the other kernel's long tiles would not pay, by what the kernel of few rows has to do at most:
// its tiles times the keys that one sees, a tile's start and end being as long as some 136 keys, times the elements of a head. A prompt of
// 128 tokens 7.5 us against 22 with its keys opened, 6 of up to 523 behind a window of 21 11 against 57, 4 of 128 behind 1000 keys 19 against
// 40; beyond it 1 of 1024 44 against 38, 1 of 2000 behind a window of 100 48 against 38, 64 tokens behind 8192 keys 54 against 47.
constexpr double kSmall = 0x1p20 * 128;
constexpr int kTileKeys = 136;
// kLeast, kOver: blocks of a piece at least and what a piece costs beside them, in blocks. Half and twice as many blocks made no difference; with
// half the cost 64 requests of up to 12 tokens, 2000 keys, took 66 us against 41, with twice 64 x 8192 tokens with heads of 256 225 against 194.
constexpr int kWaves = 4, kBlock = 32, kLeast = 8, kOver = 6;

// Workgroups a CU, by registers (blocks of 32 elements in a row). 64 x 8192 tokens, heads of 128, take 90 us with one and 76 with three; 32 x 4096
// with heads of 96 take 32 with two and 29 with three; heads of 256 spill with two, 64 x 8192 tokens 223 against 197 with one. Four of up to
// 64 elements: 46 against 48 there, but 29 against 26 for 64 x 1 tokens of 32 heads on one.
constexpr int per_cu(int blocks) { return blocks <= 4 ? 3 : blocks <= 7 ? 2 : 1; }

template <int NG> struct Shape4 {
    static constexpr int DIM = 32 * NG, ROWS = 16;
    // a piece of sixteen places in LDS: copies of 1024 bytes, the last of 256 where that is enough
    static constexpr int BYTES_IN = 288 * NG, WHOLE = BYTES_IN / 1024, TAIL = BYTES_IN % 1024, COPIES = WHOLE + (TAIL > 0);
    static constexpr int PIECE = WHOLE * 1024 + (TAIL == 0 ? 0 : TAIL <= 256 ? 256 : 1024);
    static constexpr int SLOT = 4 * PIECE;  // a block's two pieces of keys and two of values
    static constexpr int OSTRIDE = DIM + 4;  // floats between rows of a wave's results
    static constexpr int OUT = ROWS * (OSTRIDE * 4 + 8);
    static constexpr int WAVE = SLOT > OUT ? SLOT : OUT;
    static constexpr int BYTES = kWaves * WAVE;
};

__device__ __forceinline__ f4 mma16(u32x4 a, u32x4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(a8h, a), __builtin_bit_cast(a8h, b), c, 0, 0, 0);
}
// Maximum and sum over the four lanes that hold one row.
__device__ __forceinline__ float row_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return half_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}
__device__ __forceinline__ float row_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return half_sum(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}

// The f16 operand c - 8 of a dword's eight codes: nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7. (The constants are hidden, so that they stay
// in registers: an instruction that masks and sets takes no constants of its own.)
struct Open8 {
    uint32_t even_bits, even_one, odd_bits, odd_one;
    __device__ __forceinline__ void init() {
        even_bits = 0x000F000Fu, odd_bits = 0x00F000F0u, even_one = 0x64006400u, odd_one = 0x54005400u;
        asm("" : "+s"(even_bits), "+s"(odd_bits));
        asm("" : "+v"(even_one), "+v"(odd_one));
    }
    __device__ __forceinline__ u32x4 operator()(uint32_t y) const {
        const uint32_t z = y >> 8;
        const h2 a = {(_Float16)-1032.0f, (_Float16)-1032.0f}, b = {(_Float16)-72.0f, (_Float16)-72.0f};
        auto even = [&](uint32_t x) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (x & even_bits) | even_one) + a); };
        auto odd = [&](uint32_t x) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (x & odd_bits) | odd_one) + b); };
        return (u32x4){even(y), odd(y), even(z), odd(z)};
    }
};

// N dwords of LDS, W at a time.
template <int N, int W> __device__ __forceinline__ void read_lds(uint32_t (&v)[N], uint32_t at) {
    typedef uint32_t vec __attribute__((ext_vector_type(W)));
    typedef const __attribute__((address_space(3))) vec *lp;
#pragma unroll
    for (int i = 0; i < N; i += W) {
        if constexpr (W == 1) {
            typedef const __attribute__((address_space(3))) uint32_t *up;
            v[i] = *(up)(at + 4 * i);
        } else {
            const vec x = *(lp)(at + 4 * i);
#pragma unroll
            for (int j = 0; j < W; j++) v[i + j] = x[j];
        }
    }
}
__device__ __forceinline__ float half_lo(uint32_t v) { return (float)__builtin_bit_cast(h2, v)[0]; }
__device__ __forceinline__ float half_hi(uint32_t v) { return (float)__builtin_bit_cast(h2, v)[1]; }

// A piece of sixteen places of one plane in a lane: its codes and the scales of its four places, [block][place].
template <int NG> struct Piece4 {
    uint32_t codes[NG], scales[2 * NG];
    __device__ __forceinline__ void read(uint32_t at, uint32_t scales_at) {  // this lane's part of the codes, its quarter's of the scales
        read_lds<NG, NG % 4 == 0 ? 4 : NG % 2 == 0 ? 2 : 1>(codes, at);
        read_lds<2 * NG, NG % 2 == 0 ? 4 : 2>(scales, scales_at + 256 * NG);
    }
    __device__ __forceinline__ float scale(int b, int i) const {
        const uint32_t v = scales[2 * b + (i >> 1)];
        return i & 1 ? half_hi(v) : half_lo(v);
    }
};

template <int NG> struct Acc4 {
    f4 o[NG][2];
    float m, f, l;  // reference (log2 units, with the lift and the scales'); the score it came from; this lane's share of the sum
    float most;     // the highest reference so far
    bool far;
};

template <int NG, bool BF> __global__ __launch_bounds__(64 * kWaves, per_cu(NG)) void attn4_few(const AttnArgs p) {
    using S = Shape4<NG>;
    constexpr bool TWO = !BF;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), c = lane & 15, quarter = lane >> 4;
    Item it;
    if (!find_item<S::ROWS, kBlock, kLeast, kOver>(p, blockIdx.x, gridDim.x, it)) return;
    const int *table = p.table + (int64_t)it.req * p.max_pages;
    const int keys = it.kv;
    const int r0 = it.tile * S::ROWS, left = it.nq * p.group - r0, n = left < S::ROWS ? left : S::ROWS;
    // masks: this lane's rows, then the extremes over the tile
    const int first = keys - it.nq;
    auto low = [&](int hi) { return p.window > 0 && hi >= p.window ? hi - p.window + 1 : 0; };
    const int my_hi = first + p.by_group(r0 + (c < n ? c : n - 1)), my_lo = low(my_hi);
    const int hi_min = uni(first + p.by_group(r0)), hi_max = uni(first + p.by_group(r0 + n - 1)), lo_min = uni(low(hi_min)), lo_max = uni(low(hi_max));
    const Span sp = span_of<kBlock>(hi_max, lo_min, p.sinks);
    const int nb = sp.count(), piece = it.nsplit == 1 ? nb : (nb + it.nsplit - 1) / it.nsplit;
    const int b0 = it.split * piece, b1 = b0 + piece < nb ? b0 + piece : nb;

    // q in f16 operands, scaled by a power of two to at most 2^15
    u32x4 q[NG];
    float sc;
    {
        const int row = r0 + (c < n ? c : 0), t = p.by_group(row), g0 = row - t * p.group;
        const uint16_t *src = p.q + (int64_t)(it.q0 + t) * p.q_stride + (int64_t)(it.head * p.group + g0) * p.dim + 8 * quarter;
        uint4 raw[NG];
#pragma unroll
        for (int g = 0; g < NG; g++) __builtin_memcpy(&raw[g], src + 32 * g, 16);  // (rows need be aligned to their type only)
        float top = 0.0f;
        auto each = [&](int g, auto use) {
            const uint32_t x[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
            for (int i = 0; i < 4; i++) use(i, wide_lo<BF>(x[i]), wide_hi<BF>(x[i]));
        };
#pragma unroll
        for (int g = 0; g < NG; g++) each(g, [&](int, float a, float b) { top = fmaxf(top, fmaxf(fabsf(a), fabsf(b))); });
        top = row_max(top);
        int e = 141 - (int)(__float_as_uint(top) >> 23);
        e = e > 126 ? 126 : e;
        const float up = __uint_as_float((uint32_t)(e + 127) << 23);
        // (finite, while scores that fp32 holds can need more, from small keys: infinity times a difference of 0 would be NaN, and such scores
        // are so far apart that a smaller factor leaves one key all the weight too)
        sc = fminf(ldexpf(p.scale, -e), 3.4028234663852886e38f);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            each(g, [&](int i, float a, float b) { q[g][i] = __builtin_bit_cast(uint32_t, (h2){(_Float16)(a * up), (_Float16)(b * up)}); });
        }
    }

    // Where the pieces lie: a lane has the byte offset of one of the next 64 pieces that this wave takes (two a block), negative for one that
    // no row sees or whose page is out of range, and past the last block. (As scalars, piece by piece, they took half as many instructions
    // as all the rest of a block.)
    auto key_of = [&](int b) { return kBlock * sp.block(b); };
    uint32_t off_lo = 0, off_hi = 0;
    auto place = [&](int i) {  // from the wave's i-th block on
        const int b = b0 + w + (i + (lane >> 1)) * kWaves, t = key_of(b < b1 ? b : b0) + 16 * (lane & 1);
        const bool some = b < b1 && t <= hi_max && !(p.sinks <= t && lo_min >= t + 16);
        const int page = some ? table[t >> p.page_log2] : -1;
        int64_t off = (int64_t)page * p.page_bytes + (int64_t)it.head * p.head_bytes + (int64_t)((t & ((1 << p.page_log2) - 1)) >> 4) * (9 * S::DIM);
        if ((uint32_t)page >= (uint32_t)p.npages) off = -1;
        off_lo = (uint32_t)off, off_hi = (uint32_t)(off >> 32);
    };
    struct Where {
        uint32_t lo, hi, bytes;
    };
    auto where_of = [&](int i, int half) {
        const int at = (2 * i + half) & 63;
        Where x = {(uint32_t)__builtin_amdgcn_readlane((int)off_lo, at), (uint32_t)__builtin_amdgcn_readlane((int)off_hi, at), 0};
        x.bytes = (uint32_t)(9 * S::DIM) & ~(uint32_t)((int)x.hi >> 31);
        return x;
    };
    const uint32_t slot = lds_addr(lds) + w * S::WAVE, voff = 16 * lane, voff4 = 4 * lane;
    auto copy = [&](const uint8_t *plane, const Where &at, uint32_t to) {
        const dma_rsrc d = dma_desc(plane + (int64_t)(((uint64_t)at.hi << 32) | at.lo), at.bytes);
#pragma unroll
        for (int i = 0; i < S::COPIES; i++) {
            if (i < S::WHOLE || S::TAIL > 256) dma16(d, to + 1024 * i, voff, 1024 * i);
            else dma4(d, to + 1024 * i, voff4, 1024 * i);
        }
    };
    // Copies in flight behind the ones of a block's keys (or values): those of its values (or of the next block's keys).
    constexpr int AHEAD = 2 * S::COPIES;
    place(0);
    {
        const Where at[2] = {where_of(0, 0), where_of(0, 1)};
#pragma unroll
        for (int h = 0; h < 2; h++) copy(p.k, at[h], slot + h * S::PIECE);
#pragma unroll
        for (int h = 0; h < 2; h++) copy(p.v, at[h], slot + (2 + h) * S::PIECE);
    }

    Open8 open8;
    open8.init();
    Acc4<NG> A;
    A.m = A.f = A.most = -__builtin_inff();
    A.l = 0.0f;
    A.far = false;
#pragma unroll
    for (int g = 0; g < NG; g++) A.o[g][0] = A.o[g][1] = (f4){0, 0, 0, 0};
    int tl = -24;              // the scales of the values that this lane's row has seen are at most 2^tl,
    uint32_t limit = 0x0001u;  // in f16, below infinity's bits: of the row that has seen the smallest

    int turn = 1;  // the wave's block whose copies are next
    for (int b = b0 + w; b < b1; b += kWaves, turn++) {
        const int t = key_of(b);
        if ((turn & 31) == 0) place(turn);
        const Where next[2] = {where_of(turn, 0), where_of(turn, 1)};
        Piece4<NG> k[2], v[2];
        const uint32_t at = slot + 4 * NG * lane, scales_at = slot + 8 * NG * quarter;
        wait_vmcnt(AHEAD);
#pragma unroll
        for (int h = 0; h < 2; h++) k[h].read(at + h * S::PIECE, scales_at + h * S::PIECE);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the keys' part of the slot has been read
#pragma unroll
        for (int h = 0; h < 2; h++) copy(p.k, next[h], slot + h * S::PIECE);
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const f4 d = mma16(open8(k[h].codes[g]), q[g], (f4){0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * h + i] = fmaf(k[h].scale(g, i), d[i], g == 0 ? 0.0f : x[4 * h + i]);
            }
        wait_vmcnt(AHEAD);
#pragma unroll
        for (int h = 0; h < 2; h++) v[h].read(at + (2 + h) * S::PIECE, scales_at + (2 + h) * S::PIECE);
        // the scales of the values, a few a lane: larger ones than so far, and ones that are not finite
        uint32_t big = 0;
#pragma unroll
        for (int i = lane; i < 16 * NG; i += 64) {
            typedef const __attribute__((address_space(3))) uint32_t *up;
            const int h = i >= 8 * NG, j = i - h * 8 * NG;
            const uint32_t a = *(up)(slot + (2 + h) * S::PIECE + 256 * NG + 4 * j) & 0x7FFF7FFFu;
            big = big > (a & 0xFFFFu) ? big : a & 0xFFFFu;
            big = big > (a >> 16) ? big : a >> 16;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the values' part has been read
#pragma unroll
        for (int h = 0; h < 2; h++) copy(p.v, next[h], slot + (2 + h) * S::PIECE);
        const bool all = t + kBlock - 1 <= hi_min && (t >= lo_max || t + kBlock <= p.sinks);
        if (__any(big > limit)) {
            // (The pieces come whole, and what a place that a row does not see holds must not reach the row, its scale's size neither: beside
            // a hidden scale of 7936 the largest weight times a scale of 2^-10 would stand as low as 2^-16, where f16's step is 2^-24.)
            auto seen = [&](int i) {
                const int key = t + 16 * (i >> 2) + 4 * quarter + (i & 3);
                return key <= my_hi && (key >= my_lo || key < p.sinks);
            };
            if (__any(big >= 0x7C00u)) {
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    bool bad = false;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        uint32_t &d = v[i >> 2].scales[2 * g + ((i & 3) >> 1)];
                        const int sh = 16 * (i & 1);
                        if ((d >> sh & 0x7FFFu) >= 0x7C00u) {
                            bad = bad || seen(i);
                            d &= ~(0xFFFFu << sh);
                        }
                    }
                    const float nan = row_max(bad ? 1.0f : 0.0f) > 0.0f ? __builtin_nanf("") : 0.0f;
                    A.o[g][0] += nan;
                    A.o[g][1] += nan;
                }
            }
            // The largest that the row sees: of all places, or of the eight that this lane has the row's scores of.
            // (f16's bits as fp32's: exact, subnormal ones too)
            uint32_t finite = big;
            if (!all || __any(big >= 0x7C00u)) {
                finite = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    uint32_t u = 0;
#pragma unroll
                    for (int g = 0; g < NG; g++) {
                        const uint32_t d = v[i >> 2].scales[2 * g + ((i & 3) >> 1)] >> (16 * (i & 1)) & 0x7FFFu;
                        u = u > d ? u : d;
                    }
                    u = seen(i) ? u : 0;
                    finite = finite > u ? finite : u;
                }
                finite = __float_as_uint(row_max(__uint_as_float(finite << 13) * 0x1p112f));
            } else {
                finite = __builtin_amdgcn_readlane(scan64((int)finite, 0, [](int a, int b) { return a > b ? a : b; }), 63);
                finite = __float_as_uint(__uint_as_float(finite << 13) * 0x1p112f);
            }
            const float top = __uint_as_float(finite);
            const bool more = top > ldexpf(1.0f, tl);
            if (__any(more)) {
                const uint32_t u = __float_as_uint(top);
                const int to = more ? (int)(u >> 23) - 127 + ((u & 0x7FFFFFu) != 0) : tl, by = to - tl;
                tl = to;
                const int least = __builtin_amdgcn_readlane(scan64(tl, 0x7FFF, [](int a, int b) { return a < b ? a : b; }), 63);
                limit = least > 15 ? 0x7BFFu : __builtin_bit_cast(uint16_t, (_Float16)ldexpf(1.0f, least));
                const float less = ldexpf(1.0f, -by);
                A.m += (float)by;
                A.most += (float)by;
                A.l *= less;
#pragma unroll
                for (int g = 0; g < NG; g++) A.o[g][0] *= less, A.o[g][1] *= less;
            }
        }
        float least = x[0], top = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]), least = fminf(least, x[i]);
        if (__any(top == __builtin_inff() || least == -__builtin_inff())) {  // a key's scale is infinite: its score is NaN
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = fmaf(x[i], 0.0f, x[i]);
            top = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
        }
        if (!all) {
            const int from = t + 4 * quarter, dh = my_hi - from, dl = my_lo - from, ds = p.sinks - from;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = 16 * (i >> 2) + (i & 3);
                x[i] = e <= dh && (e >= dl || e < ds) ? x[i] : -__builtin_inff();
            }
            top = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
        }
        top = row_max(top);
        // The reference, as in softmax_step: raised to the largest score where that exceeds it by more than 2^8, lowered (by 2^64 in
        // all at most) to a block whose largest weight is below 2^-14. Weights stand 2^7 above it, in units of the largest scale.
        const float d = (top - A.f) * sc, lift = 7.0f - (float)tl;
        const bool fall = d < -14.0f && top > -__builtin_inff() && !A.far && A.m > A.most - 64.0f;
        if (__any(d > (A.far ? 0.0f : 8.0f) || fall)) {
            const bool move = d > (A.far ? 0.0f : 8.0f) || fall;
            float y = top * sc;
            const float bottom = A.most - 64.0f + lift;
            const bool cut = fall && y < bottom;
            y = cut ? bottom : y;
            const float from = cut ? bottom * __builtin_amdgcn_rcpf(sc) : top;
            const bool far = fabsf(y) > kFar;
            const float r = (far ? y : ceilf(y)) - lift;
            const float a = move ? exp2_hw(far && A.far ? (A.f - from) * sc : A.m - r) : 1.0f;  // from -Inf: 0
            A.l *= a;
#pragma unroll
            for (int g = 0; g < NG; g++) A.o[g][0] *= a, A.o[g][1] *= a;
            A.m = move ? r : A.m;
            A.f = move ? from : A.f;
            A.far = move ? far : A.far;
            A.most = fmaxf(A.most, A.m);
        }
        const float neg = A.far ? lift : A.m == -__builtin_inff() ? 0.0f : -A.m;
        if (__any(A.far)) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] -= A.far ? A.f : 0.0f;
        }
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = exp2_hw(fmaf(x[i], sc, neg));
            l += x[i];
        }
        A.l += l;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const u32x4 y = open8(v[0].codes[g]), z = open8(v[1].codes[g]), a0 = {y.x, y.z, z.x, z.z}, a1 = {y.y, y.w, z.y, z.w};
            u32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int h = i >> 1, j = 2 * (i & 1);
                const float e0 = x[4 * h + j], e1 = x[4 * h + j + 1], d0 = v[h].scale(g, j), d1 = v[h].scale(g, j + 1);
                hi[i] = __builtin_bit_cast(uint32_t, (h2){(_Float16)fmaf(e0, d0, 0.0f), (_Float16)fmaf(e1, d1, 0.0f)});  // (fused: with the rounding in one instruction)
                // (hidden: the compiler would round the products anew for the second term, in another way)
                if (TWO) hi[i] = hide(hi[i]);
                const h2 f = __builtin_bit_cast(h2, (uint32_t)hi[i]);
                if (TWO) lo[i] = __builtin_bit_cast(uint32_t, (h2){(_Float16)fmaf(e0, d0, -(float)f[0]), (_Float16)fmaf(e1, d1, -(float)f[1])});
            }
            A.o[g][0] = mma16(a0, hi, A.o[g][0]);
            A.o[g][1] = mma16(a1, hi, A.o[g][1]);
            if (TWO) {
                A.o[g][0] = mma16(a0, lo, A.o[g][0]);
                A.o[g][1] = mma16(a1, lo, A.o[g][1]);
            }
        }
    }
    wait_vmcnt(0);
    // the four waves' results, through LDS: rows, then references and sums
    float *mine = lds + w * (S::WAVE / 4);
    auto ml = [&](int u) { return reinterpret_cast<float2 *>(lds + u * (S::WAVE / 4) + S::ROWS * S::OSTRIDE); };
    const float l = row_sum(A.l);
    if (c < n) {
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const f4 a = A.o[g][0], b = A.o[g][1];
            float *dst = mine + c * S::OSTRIDE + 32 * g + 8 * quarter;
            *reinterpret_cast<float4 *>(dst) = make_float4(a[0], b[0], a[1], b[1]);
            *reinterpret_cast<float4 *>(dst + 4) = make_float4(a[2], b[2], a[3], b[3]);
        }
        if (quarter == 0) ml(w)[c] = make_float2(A.m, l);
    }
    __syncthreads();
    const bool direct = it.nsplit == 1;
    for (int idx = tid; idx < n * (S::DIM / 4); idx += 64 * kWaves) {
        const int r = idx / (S::DIM / 4), d = (idx - r * (S::DIM / 4)) * 4, row = r0 + r, tok = p.by_group(row);
        Join j;
        j.init();
#pragma unroll
        for (int u = 0; u < kWaves; u++) {
            const float4 o = *reinterpret_cast<const float4 *>(lds + u * (S::WAVE / 4) + r * S::OSTRIDE + d);
            const float2 y = ml(u)[r];
            j.add(y.x, y.y, o.x, o.y, o.z, o.w);
        }
        if (direct) {
            put4<BF>(p, it.q0, row, it.head, d, j.o, j.l, keys - it.nq + tok >= 0);
        } else {
            float *dst = p.part + ((int64_t)it.slot * S::ROWS + r) * (S::DIM + 2);
            agent_store(dst + d, j.o[0], j.o[1]);
            agent_store(dst + d + 2, j.o[2], j.o[3]);
            if (d == 0) agent_store(dst + S::DIM, j.m, j.l);
        }
    }
    if (direct) return;
    if (last_piece(p, it, reinterpret_cast<int *>(lds)))
        join_tile<S::DIM, S::ROWS, BF, kWaves>(p, it, r0, n, lds + 4, S::BYTES - 16);
}

template <int NG, bool BF> int launch_few(trhip_ctx *ctx, const AttnArgs &p, int64_t grid) {
    const void *fn = reinterpret_cast<const void *>(attn4_few<NG, BF>);
    const int st = allow_dyn_lds(ctx, fn, Shape4<NG>::BYTES, "kv4_attn");
    if (st != TRHIP_OK) return st;
    hipLaunchKernelGGL((attn4_few<NG, BF>), dim3((unsigned)grid), dim3(64 * kWaves), (Shape4<NG>::BYTES), ctx->stream, p);
    return launch_check(ctx, "kv4_attn");
}
int launch_few(trhip_ctx *ctx, const AttnArgs &p, bool bf, int64_t grid) {
    switch (p.dim / 32) {
    case 1: return bf ? launch_few<1, true>(ctx, p, grid) : launch_few<1, false>(ctx, p, grid);
    case 2: return bf ? launch_few<2, true>(ctx, p, grid) : launch_few<2, false>(ctx, p, grid);
    case 3: return bf ? launch_few<3, true>(ctx, p, grid) : launch_few<3, false>(ctx, p, grid);
    case 4: return bf ? launch_few<4, true>(ctx, p, grid) : launch_few<4, false>(ctx, p, grid);
    case 5: return bf ? launch_few<5, true>(ctx, p, grid) : launch_few<5, false>(ctx, p, grid);
    case 6: return bf ? launch_few<6, true>(ctx, p, grid) : launch_few<6, false>(ctx, p, grid);
    case 7: return bf ? launch_few<7, true>(ctx, p, grid) : launch_few<7, false>(ctx, p, grid);
    default: return bf ? launch_few<8, true>(ctx, p, grid) : launch_few<8, false>(ctx, p, grid);
    }
}

}  // namespace

int launch_kv4_attn(trhip_ctx *ctx, const trhip_kv4 *kv, const AttnCall &c, int io) {
    AttnArgs p = {};
    p.q = static_cast<const uint16_t *>(c.q);
    p.out = static_cast<uint16_t *>(c.out);
    p.q_stride = c.q_stride;
    p.out_stride = c.out_stride;
    p.k = static_cast<const uint8_t *>(kv->k);
    p.v = static_cast<const uint8_t *>(kv->v);
    p.head_bytes = kv->page * kv->dim / 16 * 9;
    p.page_bytes = (int64_t)p.head_bytes * kv->heads;
    p.npages = kv->pages;
    p.page_log2 = __builtin_ctz((unsigned)kv->page);
    p.table = c.table;
    p.max_pages = c.max_pages;
    p.q_start = c.q_start;
    p.kv_len = c.kv_len;
    p.nreq = (int)c.nreq;
    p.tokens = (int)c.tokens;
    p.heads = c.heads;
    p.kv_heads = kv->heads;
    p.group = c.heads / kv->heads;
    p.dim = kv->dim;
    p.window = (int)c.window;
    p.sinks = (int)c.sinks;
    p.scale = c.scale * 1.44269504088896341f;
    p.by_group.of(p.group);
    p.by_heads.of(p.kv_heads);
    p.out_aligned = (reinterpret_cast<uintptr_t>(c.out) % 8 == 0) && c.out_stride % 4 == 0;
    p.arrivals = ctx->arrivals;
    const int cus = ctx->sm_count > 0 ? ctx->sm_count : 256;
    const int64_t most_new = c.max_new < c.tokens ? c.max_new : c.tokens;
    // Requests of more than kTokMost rows: their keys go to the workspace in 16 bits and the 16-bit cache's kernel of many rows takes
    // them, where the workspace may hold the longest ones that the sizes allow. Which there are is known only from the hint.
    const int64_t most_long = c.tokens * p.group / (kTokMost + 1), longs = most_long < c.nreq ? most_long : c.nreq;
    const double cap = (double)c.max_pages * kv->page, window = (double)c.window + (double)c.sinks + 16, seen = c.window > 0 && window < cap ? window : cap;
    const double tiles = ((double)c.tokens * p.group / 16 + (double)c.nreq) * kv->heads;
    const double image_bytes = (double)longs * (double)c.max_pages * (double)p.page_bytes * (32.0 / 9.0);
    bool image = most_new * p.group > kTokMost && tiles * (seen + kTileKeys) * kv->dim > kSmall && longs > 0 && longs < 65536 && p.kv_heads < 65536 && c.max_pages > 0 && image_bytes <= (double)kMostImage &&
                       (double)c.nreq * (double)c.max_pages <= (double)(kMostImage / 4);
    const int64_t plane = image ? (longs * c.max_pages * (p.page_bytes / 9 * 32) + 255) & ~(int64_t)255 : 0, tables = image ? c.nreq * c.max_pages * 4 : 0;
    uint8_t *room = nullptr;
    // (no memory for it: the kernel of few rows takes all requests, and does so in a capture behind such a call)
    if (image && ctx->no_room && (size_t)(2 * plane + tables) >= ctx->no_room && capturing(ctx)) image = false;
    if (image) {
        int st = TRHIP_OK;
        room = static_cast<uint8_t *>(workspace2(ctx, (size_t)(2 * plane + tables), &st));
        if (!room && st != TRHIP_ERR_OOM) return st;
        image = room != nullptr;
        ctx->no_room = image ? 0 : (size_t)(2 * plane + tables);
    }
    p.row_lo = 0;
    p.row_hi = image ? kTokMost : kAnyRows;
    const int rows = 16;
    p.target = cus * per_cu(kv->dim / 32);
    const int64_t grid = plan_items(p, c, rows, kBlock, kLeast);
    // (workgroups times threads has to stay below 2^32)
    if (grid >= ((int64_t)1 << 32) / (64 * kWaves)) return fail(ctx, TRHIP_ERR_INVALID, "kv4_attn: too many rows");
    if (image) {
        int st = TRHIP_OK;
        const Image4 im = {p.k, p.v, reinterpret_cast<uint16_t *>(room), reinterpret_cast<uint16_t *>(room + plane), reinterpret_cast<int *>(room + 2 * plane),
                           p.q_start, p.kv_len, p.table, p.max_pages, p.npages, p.nreq, p.tokens, p.group, p.kv_heads, p.dim, p.page_log2, kTokMost,
                           p.window, p.sinks, io == TRHIP_BF16};
        st = launch_attn4_image(ctx, im, (int)longs);
        if (st != TRHIP_OK) return st;
        const trhip_kv open = {io, kv->page, kv->heads, kv->dim, longs * c.max_pages, room, room + plane};
        AttnCall lc = c;
        lc.table = im.out_table;
        lc.long_only = true;
        st = launch_attn(ctx, &open, lc);
        if (st != TRHIP_OK) return st;
    }
    int st = TRHIP_OK;
    float *ws = static_cast<float *>(workspace(ctx, (size_t)p.part_slots * rows * (kv->dim + 2) * sizeof(float), &st));
    if (!ws) return st;
    p.part = ws;
    return launch_few(ctx, p, io == TRHIP_BF16, grid);
}

}  // namespace trhip
