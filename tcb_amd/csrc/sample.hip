// sample.hip -- the next token of each row of logits: temperature, top-k, top-p and min-p, from a given random number.
//
// Two launches; the first reads every logit once. A row is cut into stripes of 256 entries, dealt in turn to the waves of its
// workgroups, which hold them in registers. A workgroup leaves, as the row's settings need it,
//   the weight of each of its stripes, relative to its own largest logit (rows without a filter, and the sum that top_p is a part of),
//   its largest entries, by a threshold that at least as many of its threads' maxima reach (rows with a filter),
//   its weights in bins of a ninety-sixth of a nat (top_p without top_k).
// The second, a workgroup a row, finishes it: without a filter it finds the stripe in which the random number falls, and there the
// entry; with one it takes the entries that the workgroups left (some hundreds), cuts the run that is kept, and walks it by index. The
// workgroups' shares are what a row whose large entries lie anywhere needs with room to spare; whether they are complete is checked, and a row
// where they are not (a flat one, of which thousands are kept, or one whose largest entries lie in few stripes) is read again, a few
// times: the bin in which the run ends is opened until its entries can be sorted (at once, where its weight says that they are few), then all
// stripes are weighed.
//
// Weights and their sums are in 64 bits, since one border among a hundred thousand has to be met: e^x by a table of 64 powers and a
// polynomial of degree 5.
//
// 1 x 128256, fp32: 10 us without a filter, 13 with top_k 50, 16 with top_p .85 (two launches, the second one's chain of steps by one workgroup);
// a flat row of which thousands are kept 91 to 94, by one CU that reads the row once more. 256 x 128256, from memory: 37 us for the largest, 53 without
// a filter, 45 with top_k 50, 84 with top_p .85 of peaked rows and 148 where some keep thousands. In the first launch 32 (4.2 TB/s), 51 (a 64-bit
// exponential of every logit), 41 (the threshold, after all of a workgroup's loads), 87 (bins in LDS by 64-bit atomics); the second takes 6 to 7,
// and 70 of those 148.
#include "trhip_internal.hpp"

namespace trhip {
namespace {

constexpr int kRead = 512, kEnd = 1024;  // threads of the two launches
constexpr int kStripe = 256, kMost = 1024;  // kMost: entries that are sorted at most
constexpr int kBins = 2048;
constexpr float kPerNat = 96.0f;

struct SampleArgs {
    const void *logits;
    int io;
    int64_t stride;
    int vocab, stripes, groups, room;  // room: entries that a workgroup may leave
    int wide;                          // four entries at a time
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    int *token;
    float *logprob;
    double *mass;           // [row][stripe]
    unsigned long long *list;  // [row][workgroup][room]: key, ~index
    unsigned long long *hist;  // [row][workgroup][kBins]: weight in bins of its logits, from the largest's down (bin_exponent)
    uint4 *left;               // [row][workgroup]: largest key, threshold (0: all entries left), entries left
};

// A logit as an unsigned number in the same order; NaN and -Inf are 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    if (!(x > -__builtin_inff())) return 0;
    if (b == 0x80000000u) return 0x80000000u;  // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

struct Row {
    const void *x;
    int io, vocab, wide;
    __device__ __forceinline__ float value(int i) const {
        return io == TRHIP_F32 ? static_cast<const float *>(x)[i] : h16_to_f32(static_cast<const uint16_t *>(x)[i], io);
    }
    __device__ __forceinline__ uint32_t key(int i) const { return key_of(value(i)); }
    // entries i .. i + 3 (i a multiple of 4); NaN past the last
    __device__ __forceinline__ void values4(int i, float (&f)[4]) const {
        if (wide && i + 4 <= vocab) {
            if (io == TRHIP_F32) {
                *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
            } else {
                const uint2 y = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(x) + i);
                f[0] = h16_to_f32(y.x & 0xFFFFu, io), f[1] = h16_to_f32(y.x >> 16, io);
                f[2] = h16_to_f32(y.y & 0xFFFFu, io), f[3] = h16_to_f32(y.y >> 16, io);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; u++) f[u] = i + u < vocab ? value(i + u) : __builtin_nanf("");
        }
    }
    // and their keys, 0 past the last
    __device__ __forceinline__ void keys4(int i, uint32_t (&k)[4]) const {
        float f[4];
        values4(i, f);
#pragma unroll
        for (int u = 0; u < 4; u++) k[u] = key_of(f[u]);
    }
    // This lane's entries of stripes first, first + apart, ..., N of them. Where the row has them whole no load is behind a condition, or
    // the next one would wait for it.
    template <int N> __device__ __forceinline__ void stripes(int first, int apart, float (&f)[N][4]) const {
        const int i = first * kStripe + 4 * (int)(threadIdx.x & 63), step = apart * kStripe;
        const bool in = wide && (first + (N - 1) * apart + 1) * kStripe <= vocab;
        if (in && io == TRHIP_F32) {
#pragma unroll
            for (int a = 0; a < N; a++) *reinterpret_cast<float4 *>(f[a]) = *reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i + a * step);
        } else if (in) {
            uint2 y[N];
#pragma unroll
            for (int a = 0; a < N; a++) y[a] = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(x) + i + a * step);
#pragma unroll
            for (int a = 0; a < N; a++) {
                f[a][0] = h16_to_f32(y[a].x & 0xFFFFu, io), f[a][1] = h16_to_f32(y[a].x >> 16, io);
                f[a][2] = h16_to_f32(y[a].y & 0xFFFFu, io), f[a][3] = h16_to_f32(y[a].y >> 16, io);
            }
        } else {
#pragma unroll
            for (int a = 0; a < N; a++) values4(i + a * step < vocab ? i + a * step : vocab, f[a]);
        }
    }
};

// e^((l - max) / T) of a logit or its key; 0 of NaN and -Inf, 1 of +Inf (max is 1e300 then, and 1 / T
// is not quite 0, so that an infinite temperature leaves an infinite logit alone). e^t = 2^(n / 64) e^r, n = rint(64 t / ln 2),
// |r| <= ln 2 / 128: what r^6 / 720 leaves out is 2^-54. Twenty operations; t is rounded once more, which is 2^-53 |t|.
struct Weight {
    uint32_t top;
    double max, inv;
    const double *table;  // 2^(j / 64)
    __device__ __forceinline__ Weight(uint32_t top, double inv, const double *table)
        : top(top), max(top == 0xFF800000u ? 1e300 : (double)of_key(top)), inv(fmax(inv, 1e-290)), table(table) {}
    __device__ __forceinline__ double of(float f) const {
        const double t = fmin(fmax(((double)f - max) * inv, -1100.0), 0.0);
        const double z = fma(t, 92.33248261689366, 0x1.8p52), n = z - 0x1.8p52;  // z's low bits are n
        const double r = fma(-n, 3.623510646634843e-19, fma(-n, 0.010830424696249145, t));  // (ln 2 / 64 in two parts)
        double y = fma(r, 8.3333333333333332e-3, 4.1666666666666664e-2);
        y = fma(r, y, 1.6666666666666666e-1);
        y = fma(r, y, 0.5);
        y = fma(r, y, 1.0);
        const int i = (int)(uint32_t)__double_as_longlong(z);
        const double p = table[i & 63];
        return ldexp(fma(p, r * y, p), i >> 6);
    }
    __device__ __forceinline__ double operator()(uint32_t k) const { return of(of_key(k)); }
};

struct Setting {
    float t, tp, low;
    int k;  // 0: all
    bool greedy;
    double u;
};
__device__ __forceinline__ Setting setting_of(const SampleArgs &p, int r) {
    Setting s;
    s.t = p.temperature ? p.temperature[r] : 1.0f;
    s.greedy = !(s.t > 0.0f);
    s.k = s.greedy ? 1 : p.top_k ? p.top_k[r] : 0;
    if (s.k < 0 || s.k >= p.vocab) s.k = 0;
    if (s.greedy) s.k = 1;
    s.tp = s.greedy ? 1.0f : p.top_p ? p.top_p[r] : 1.0f;
    if (!(s.tp < 1.0f)) s.tp = 1.0f;
    s.low = s.greedy || !p.min_p ? 0.0f : p.min_p[r];
    if (!(s.low > 0.0f)) s.low = 0.0f;
    if (s.low > 1.0f) s.low = 1.0f;
    const float u = p.u[r];
    // (from 1 up infinite: no sum exceeds a goal of that, while the sum of all can differ from a running sum's end by a rounding)
    s.u = u >= 1.0f ? (double)__builtin_inff() : u >= 0.0f ? (double)u : 0.0;
    return s;
}
// How many entries of the whole row its workgroups should cover, and a workgroup's share of them: the mean, three standard deviations of
// entries that lie anywhere, and four. (Four and six left no room for k 293 of 1 x 128256, 32 workgroups, in the 1024 that are sorted:
// 112 us by reading again, 23 so.)
// Without top_k the run of top_p is unknown: 128 entries (with 64, 256 x 128256 of top_p .95 take 144 us against 105, with 256, 1 x 128256 takes
// 35 against 32 then).
constexpr int kCover = 128;
__device__ __forceinline__ int share_of(int n, int groups) {
    const float m = (float)n * __builtin_amdgcn_rcpf((float)groups);
    const int s = (int)(m + 3.0f * __builtin_amdgcn_sqrtf(m) + 4.0f);
    return s < n ? s : n;
}

// Bins of logits over the temperature: the number of a key's bin, which rises with it or stays. (Finite times finite: a temperature may be
// infinite or so small that its inverse is.)
__device__ __forceinline__ float bins_a_unit(float t) { return fminf(kPerNat / t, 3.4028234663852886e38f); }
__device__ __forceinline__ int bin_of(uint32_t k, float per) {
    const float f = fminf(fmaxf(of_key(k), -3.4028234663852886e38f), 3.4028234663852886e38f);
    return (int)floorf(fminf(fmaxf(f * per, -536870912.0f), 536870912.0f));
}

// Weights in a bin stand in fixed point, whose sums do not depend on the order; the unit is 2^-(48 + e) of the largest weight, e a little
// below the bin's distance from it in powers of two, so that a sum's error is that of its largest weight whatever the bin (2^-48 of it). A
// power of two is 96 ln 2 = 66.54 bins; 984 / 65536 is 1 / 66.6.
__device__ __forceinline__ int bin_exponent(int b) { return b < 2 ? 0 : ((b - 1) * 984) >> 16; }

// The nearest whole number of one up to 2^51 (the sum's last bits; a conversion is twelve instructions).
__device__ __forceinline__ unsigned long long whole(double x) {
    return (unsigned long long)__double_as_longlong(x + 0x1p52) - 0x4330000000000000ull;
}

// Inclusive sums over the wave's lanes, in six lane moves (row_shr 1, 2, 4, 8, then row_bcast 15 and 31).
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ double moved(double v) {
    const long long x = __double_as_longlong(v);
    const uint32_t lo = moved<CTRL, ROWS>((uint32_t)x), hi = moved<CTRL, ROWS>((uint32_t)(x >> 32));
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
template <class T> __device__ __forceinline__ T running(T v) {
    v += moved<0x111, 0xF>(v);
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);
    return v + moved<0x143, 0xC>(v);
}
// The lane before's value; 0 in the first.
template <class T> __device__ __forceinline__ T before_lane(T v) {
    const T up = __shfl_up(v, 1);
    return (threadIdx.x & 63) ? up : T(0);
}
__device__ __forceinline__ double of_lane(double v, int lane) {
    const long long x = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane), hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), lane);
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ double wave_sum(double v) { return of_lane(running(v), 63); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = up(v, moved<0x111, 0xF>(v));
    v = up(v, moved<0x112, 0xF>(v));
    v = up(v, moved<0x114, 0xF>(v));
    v = up(v, moved<0x118, 0xF>(v));
    v = up(v, moved<0x142, 0xA>(v));
    return of_lane(up(v, moved<0x143, 0xC>(v)), 63);
}

// ---- reading ------------------------------------------------------------------------------------------------------------

template <int J> __global__ __launch_bounds__(kRead) void sample_read(const SampleArgs p) {
    constexpr int WAVES = kRead / 64;
    __shared__ double s_table[64];
    __shared__ uint32_t s_max[kRead];
    __shared__ uint32_t s_left;
    __shared__ unsigned long long s_bins[kBins];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = blockIdx.y, g = blockIdx.x;
    const Row x = {static_cast<const char *>(p.logits) + r * p.stride * (p.io == TRHIP_F32 ? 4 : 2), p.io, p.vocab, p.wide};
    uint32_t key[J][4], top = 0;
    auto stripe = [&](int j) { return g + p.groups * (w + WAVES * j); };
    {
        float f[J][4];
        x.stripes(stripe(0), p.groups * WAVES, f);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) key[j][v] = key_of(f[j][v]);
    }
    const Setting st = setting_of(p, r);
    const bool filtered = st.k > 0 || st.tp < 1.0f || st.low > 0.0f, weigh = !filtered || (st.k == 0 && st.tp < 1.0f), bins = weigh && filtered;
    if (weigh && tid < 64) s_table[tid] = exp2((double)tid / 64.0);
    if (bins)
        for (int i = tid; i < kBins; i += kRead) s_bins[i] = 0;
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int v = 0; v < 4; v++) top = top > key[j][v] ? top : key[j][v];
    s_max[tid] = top;
    if (tid == 0) s_left = 0;
    __syncthreads();
    uint32_t mine[WAVES], least = 0xFFFFFFFFu;  // every wave has all threads' maxima
    top = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        mine[i] = s_max[64 * i + lane];
        top = top > mine[i] ? top : mine[i];
        least = least < mine[i] ? least : mine[i];
    }
    top = wave_max(top);
    uint32_t bound = 0, left = 0;
    if (weigh && top != 0) {
        const Weight wt(top, 1.0 / (double)st.t, s_table);
        const float per = bins_a_unit(st.t);
        const int first = bin_of(top, per);
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (stripe(j) >= p.stripes) break;
            double y[4];
#pragma unroll
            for (int v = 0; v < 4; v++) y[v] = wt(key[j][v]);
            if (bins) {
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int b = first - bin_of(key[j][v], per);
                    if (key[j][v] != 0 && (uint32_t)b < (uint32_t)kBins) atomicAdd(&s_bins[b], whole(ldexp(y[v], 48 + bin_exponent(b))));
                }
            }
            const double sum = wave_sum((y[0] + y[1]) + (y[2] + y[3]));
            if (lane == 0) p.mass[(int64_t)r * p.stripes + stripe(j)] = sum;
        }
    }
    if (filtered && top != 0) {
        const int share = share_of(st.k > 0 ? st.k : kCover, p.groups);
        if ((share + share / 6 + 3) * p.groups > kMost || share * 5 / 4 + 8 > p.room) {  // (too many to sort)
            left = 0xFFFFFFFFu;
        } else {
            // a threshold that `share` to share * 9 / 8 + 2 threads' maxima reach: halving between the smallest and the largest
            auto count = [&](uint32_t k) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < WAVES; i++) n += __popcll(__ballot(mine[i] >= k));
                return n;
            };
            uint32_t lo = ~wave_max(~least), hi = top;  // count(lo) >= share
            if (lo == 0 && count(1) >= share) lo = 1;
            if (lo != 0) {
                if (count(top) >= share) lo = top;
                while (lo < hi) {
                    const uint32_t mid = lo + (hi - lo + 1) / 2;
                    const int n = count(mid);
                    if (n >= share) {
                        lo = mid;
                        if (n <= share + share / 8 + 2) break;
                    } else {
                        hi = mid - 1;
                    }
                }
            }
            bound = lo;
            unsigned long long *to = p.list + ((int64_t)r * p.groups + g) * p.room;
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int v = 0; v < 4; v++) n += key[j][v] != 0 && key[j][v] >= bound;
            const uint32_t incl = running(n);
            uint32_t base = 0;
            if (lane == 63 && incl != 0) base = atomicAdd(&s_left, incl);
            uint32_t at = of_lane(base, 63) + (incl - n);
            if (n != 0) {
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        if (key[j][v] != 0 && key[j][v] >= bound) {
                            if (at < (uint32_t)p.room) to[at] = ((unsigned long long)key[j][v] << 32) | (uint32_t)~(stripe(j) * kStripe + 4 * lane + v);
                            at++;
                        }
            }
        }
    }
    __syncthreads();
    if (bins && top != 0)
        for (int i = tid; i < kBins; i += kRead) p.hist[((int64_t)r * p.groups + g) * kBins + i] = s_bins[i];
    if (tid == 0) p.left[(int64_t)r * p.groups + g] = make_uint4(top, bound, left ? left : s_left, 0);
}

// ---- finishing ------------------------------------------------------------------------------------------------------------

constexpr int kWaves = kEnd / 64;

struct Lds {
    double table[64];
    unsigned long long sorted[kMost];
    double weight[kMost];
    unsigned long long bins[kBins];
    uint32_t count[kBins];  // entries in a bin, or a workgroup's, or a stripe's
    uint32_t from[kMost];   // where a workgroup's entries go
    uint32_t u[kWaves];
    double wave[kWaves];
    uint32_t small[8];
    double sum;
};

// Over the workgroup; every thread gets the result.
__device__ __forceinline__ uint32_t all_max(uint32_t v, Lds &s) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.u[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s.u[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) v = v > s.u[w] ? v : s.u[w];
    return v;
}
// Sum over the threads before this one, and over all.
template <class T> __device__ __forceinline__ T before_me(T v, T *lds, T &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T x = running(v);
    __syncthreads();
    if (lane == 63) lds[w] = x;
    __syncthreads();
    T base = T(0);
    total = T(0);
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        if (i == w) base = total;
        total += lds[i];
    }
    return base + before_lane(x);
}
// The first thread for which `is` holds (kEnd: none).
__device__ __forceinline__ int first_of(bool is, Lds &s) {
    const uint64_t m = __ballot(is);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.u[threadIdx.x >> 6] = m ? (threadIdx.x & ~63) + __builtin_ctzll(m) : kEnd;
    __syncthreads();
    uint32_t v = s.u[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) v = v < s.u[w] ? v : s.u[w];
    return (int)v;
}
__device__ __forceinline__ int last_of(bool is, Lds &s) {
    const uint64_t m = __ballot(is);
    return (int)all_max(m ? (threadIdx.x & ~63) + 64 - __builtin_clzll(m) : 0, s) - 1;
}

// The value of lane ^ J.
template <int J> __device__ __forceinline__ uint32_t across(uint32_t v) {
    if constexpr (J == 1) return moved<0xB1, 0xF>(v);        // quads 1 0 3 2
    else if constexpr (J == 2) return moved<0x4E, 0xF>(v);   // 2 3 0 1
    else if constexpr (J == 4) return moved<0x1B, 0xF>(moved<0x141, 0xF>(v));  // eights the other way round, then quads
    else if constexpr (J == 8) return moved<0x128, 0xF>(v);  // rows of sixteen by eight
    else {
        const auto s = J == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & J ? s[0] : s[1];
    }
}
__device__ __forceinline__ void order(unsigned long long &v, unsigned long long o, bool larger) {
    const bool is = o > v;
    v = is == larger ? o : v;
}
// One step of a bitonic sort between lanes: blocks of k fall where `falling` (this thread's block) holds.
template <int J> __device__ __forceinline__ void step(unsigned long long &v, bool falling) {
    const unsigned long long o = ((unsigned long long)across<J>((uint32_t)(v >> 32)) << 32) | across<J>((uint32_t)v);
    order(v, o, ((threadIdx.x & J) == 0) == falling);
}

// The steps of blocks of k that stay within a wave.
__device__ __forceinline__ void steps(unsigned long long &v, int k, bool falling) {
    if (k >= 64) step<32>(v, falling);
    if (k >= 32) step<16>(v, falling);
    if (k >= 16) step<8>(v, falling);
    if (k >= 8) step<4>(v, falling);
    if (k >= 4) step<2>(v, falling);
    step<1>(v, falling);
}
// The wave's 64 values in order.
__device__ __forceinline__ void wave_sort(unsigned long long &v, bool falling) {
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1) steps(v, k, ((threadIdx.x & 63 & k) == 0) == falling);
}

// Sorts s.sorted[0 .. n), padded to a power of two with 0 (falling) or ~0: largest first, or smallest. A thread has an entry; steps
// within a wave move it between lanes, only those between waves go through LDS (10 of 55 for 1024 entries: 9 us with all of them).
__device__ __forceinline__ void sort(Lds &s, int n, bool falling) {
    static_assert(kEnd == kMost, "an entry a thread");
    const int tid = threadIdx.x;
    int n2 = 2;
    while (n2 < n) n2 <<= 1;
    __syncthreads();
    unsigned long long v = tid < n ? s.sorted[tid] : falling ? 0 : ~0ull;
    for (int k = 2; k <= n2; k <<= 1) {
        const bool falls = ((tid & k) == 0) == falling;
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            if (tid < n2) s.sorted[tid] = v;
            __syncthreads();
            if (tid < n2) order(v, s.sorted[tid ^ j], ((tid & j) == 0) == falls);
        }
        if ((tid & ~63) < n2) steps(v, k, falls);
    }
    __syncthreads();
    if (tid < n2) s.sorted[tid] = v;
    __syncthreads();
}

__device__ __forceinline__ void result(const SampleArgs &p, int r, int token, double w, double total) {
    p.token[r] = token;
    if (p.logprob) p.logprob[r] = (float)log(w / total);
}

// The entry of stripe `at` in which the goal falls, the weights before the stripe being `before`; by one wave. False: no entry of it has
// weight.
template <class F>
__device__ __forceinline__ bool last_stripe(const SampleArgs &p, int r, const Row &x, int at, double before, double goal, double total, F weight) {
    const int lane = threadIdx.x & 63;
    uint32_t k[4];
    x.keys4(at * kStripe + 4 * lane, k);
    double y[4], sum = 0;
#pragma unroll
    for (int v = 0; v < 4; v++) y[v] = weight(k[v], (uint32_t)(at * kStripe + 4 * lane + v)), sum += y[v];
    double run = before + before_lane(running(sum)), chosen = 0, final = 0;
    int found = -1, last = -1;
#pragma unroll
    for (int v = 0; v < 4; v++) {
        run += y[v];
        if (y[v] > 0) last = v, final = y[v];
        if (y[v] > 0 && run > goal && found < 0) found = v, chosen = y[v];
    }
    const uint64_t over = __ballot(found >= 0), some = __ballot(last >= 0);
    if (some == 0) return false;
    const int src = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
    if (lane == src) result(p, r, at * kStripe + 4 * lane + (over ? found : last), over ? chosen : final, total);
    return true;
}

// The entry in which u falls among stripes of these weights: mass(i), in one order for every call, and weight(key, index) of their entries.
template <class M, class F>
__device__ __forceinline__ void by_stripes(const SampleArgs &p, int r, const Row &x, double u, Lds &s, M mass, F weight) {
    const int tid = threadIdx.x;
    const int each = (p.stripes + kEnd - 1) / kEnd, s0 = tid * each < p.stripes ? tid * each : p.stripes, s1 = s0 + each < p.stripes ? s0 + each : p.stripes;
    double sum = 0, total;
    for (int i = s0; i < s1; i++) sum += mass(i);
    const double before = before_me(sum, s.wave, total), goal = u * total;
    int t = first_of(sum > 0 && before + sum > goal, s);
    const bool none = t == kEnd;  // u of 1 and above
    if (none) t = last_of(sum > 0, s);
    __syncthreads();
    if (tid == t) {
        double run = before, at_run = before;
        int at = s0;
        for (int i = s0; i < s1; i++) {
            const double y = mass(i);
            if (y > 0) at = i, at_run = run;
            run += y;
            if (!none && y > 0 && run > goal) break;
        }
        s.small[0] = (uint32_t)at;
        s.sum = at_run;
    }
    __syncthreads();
    if (tid >= 64) return;
    // A stripe's weight is relative to its workgroup's largest logit, and may be there where each of its entries' is below 2^-1074, which is
    // 0: then the entry is in the next stripe that has one with weight (the goal is 0: the first of all), or in the one before (the last).
    // The largest logit's is on that side.
    for (int at = (int)s.small[0]; at >= 0 && at < p.stripes; at += none ? -1 : 1)
        if (last_stripe(p, r, x, at, s.sum, goal, total, weight)) return;
}

// A filtered row whose kept run is among its largest 64 entries, by one wave: those that a threshold leaves of the n in s.sorted.
// False: it is not, or that is not certain.
__device__ __forceinline__ bool top64(const SampleArgs &p, int r, const Weight &wt, const Setting &st, double total, uint32_t complete, int n, Lds &s) {
    const int lane = threadIdx.x & 63;
    constexpr int PER = kMost / 64;
    uint32_t k[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) k[i] = 64 * i + lane < n ? (uint32_t)(s.sorted[64 * i + lane] >> 32) : 0;
    uint32_t lo = 1, hi = wt.top;  // at least `want` entries reach lo
    int count = n;
    const int want = st.k > 0 ? st.k : 40;
    if (count > 64) {
        uint32_t least = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (64 * i + lane < n) least = least < k[i] ? least : k[i];
        lo = ~wave_max(~least);
    }
    while (count > 64 && lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (i % 4 == 0 && 64 * i >= n) break;
            c += __popcll(__ballot(k[i] >= mid));
        }
        if (c >= want) lo = mid, count = c;
        else hi = mid - 1;
    }
    if (count > 64) return false;
    unsigned long long *some = s.bins;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i % 4 == 0 && 64 * i >= n) break;
        const uint64_t m = __ballot(k[i] >= lo);
        if (k[i] >= lo) some[at + __popcll(m & (((uint64_t)1 << lane) - 1))] = s.sorted[64 * i + lane];
        at += __popcll(m);
    }
    __builtin_amdgcn_wave_barrier();
    unsigned long long e = lane < count ? some[lane] : 0;
    wave_sort(e, true);
    const uint32_t key = (uint32_t)(e >> 32), index = ~(uint32_t)e;
    const bool in = lane < count && (st.k == 0 || lane < st.k);
    const double w = in ? wt(key) : 0.0, incl = running(w), before = before_lane(incl), sum = of_lane(incl, 63);
    // every entry from here up is in these lanes
    const uint32_t from = count < n && lo > complete ? lo : complete;
    const bool sure = lane < count && key >= from;
    const double goal = (double)st.tp * (st.k > 0 ? sum : total);
    const bool keep = in && (lane == 0 || ((st.tp >= 1.0f || before < goal) && w >= (double)st.low));
    const int kept = __popcll(__ballot(keep)), certain = __popcll(__ballot(sure));
    if (from != 0) {
        if (kept > certain || (kept == certain && kept != st.k)) return false;  // (the run may go on past what is here)
        if (st.k > 0 && st.tp < 1.0f && certain < st.k) return false;           // (nor is the sum certain)
    }
    // the kept ones by index, and their running sum
    unsigned long long by = lane < kept ? ((unsigned long long)index << 32) | (uint32_t)lane : ~0ull;
    wave_sort(by, false);
    const double v = __shfl(w, (int)((uint32_t)by & 63));
    const double y = lane < kept ? v : 0.0, run = running(y), kept_sum = of_lane(run, 63);
    // the first that is over the goal, or the last that has weight
    const uint64_t over = __ballot(run > st.u * kept_sum), has = __ballot(y > 0);
    if (lane == (over ? __builtin_ctzll(over) : 63 - __builtin_clzll(has))) result(p, r, (int)(by >> 32), y, kept_sum);
    return true;
}

__global__ __launch_bounds__(kEnd) void sample_end(const SampleArgs p) {
    __shared__ Lds s;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = blockIdx.x;
    const Row x = {static_cast<const char *>(p.logits) + r * p.stride * (p.io == TRHIP_F32 ? 4 : 2), p.io, p.vocab, p.wide};
    const uint4 *lefts = p.left + (int64_t)r * p.groups;
    static_assert(kEnd == kMost, "an entry, a workgroup or a stripe a thread");
    // every wave goes through all workgroups' records: the row's largest key, the key from which up every entry has been left by
    // its workgroup, how many a workgroup left at most and all together, and how many those before each one
    uint32_t top = 0, complete = 0, worst = 0, n_all = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
        uint4 left = {0, 0, 0, 0};
        if (g0 + lane < p.groups) left = lefts[g0 + lane];
        const uint32_t a = wave_max(left.x), b = wave_max(left.y), c = wave_max(left.z), n = left.z < kMost ? left.z : kMost, sum = running(n);
        top = top > a ? top : a;
        complete = complete > b ? complete : b;
        worst = worst > c ? worst : c;
        if (w == 0 && g0 + lane < p.groups) s.from[g0 + lane] = n_all + (sum - n), s.count[g0 + lane] = n;
        n_all += of_lane(sum, 63);
    }
    const Setting st = setting_of(p, r);
    const bool filtered = st.k > 0 || st.tp < 1.0f || st.low > 0.0f;
    if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
    __syncthreads();
    if (top == 0) {
        if (tid == 0) {
            p.token[r] = -1;
            if (p.logprob) p.logprob[r] = __builtin_nanf("");
        }
        return;
    }
    const Weight wt(top, st.greedy ? 1.0 : 1.0 / (double)st.t, s.table);
    const bool weighed = !filtered || (st.k == 0 && st.tp < 1.0f);
    // the workgroups' largest logits' weights, by which theirs are multiplied
    if (weighed) {
        if (tid < p.groups) {
            const uint32_t k = lefts[tid].x;
            s.weight[tid] = k ? wt(k) : 0.0;
        }
        __syncthreads();
    }
    auto mass = [&](int i) {
        const double unit = s.weight[i % p.groups];
        return unit > 0 ? p.mass[(int64_t)r * p.stripes + i] * unit : 0.0;
    };
    if (!filtered) return by_stripes(p, r, x, st.u, s, mass, [&](uint32_t key, uint32_t) { return wt(key); });
    double total = 0;
    if (weighed) {
        double sum = 0;
        for (int i = tid; i < p.stripes; i += kEnd) sum += mass(i);
        before_me(sum, s.wave, total);
    }
    bool done = false;
    if (worst <= (uint32_t)p.room && n_all <= kMost) {
        const int n = (int)n_all;
        // (a wave a workgroup's entries; two at a time, so that their loads are in flight together)
        for (int g = w; g < p.groups; g += 2 * kWaves) {
            const int g1 = g + kWaves < p.groups ? g + kWaves : g;
            const uint32_t n0 = s.count[g], n1 = g1 != g ? s.count[g1] : 0, f0 = s.from[g], f1 = s.from[g1];
            const unsigned long long *l0 = p.list + ((int64_t)r * p.groups + g) * p.room, *l1 = p.list + ((int64_t)r * p.groups + g1) * p.room;
            for (uint32_t i = lane; i < (n0 > n1 ? n0 : n1); i += 64) {
                const unsigned long long e0 = i < n0 ? l0[i] : 0, e1 = i < n1 ? l1[i] : 0;
                if (i < n0) s.sorted[f0 + i] = e0;
                if (i < n1) s.sorted[f1 + i] = e1;
            }
        }
        __syncthreads();
        if (st.k <= 64) {
            if (w == 0) {
                const bool is = top64(p, r, wt, st, total, complete, n, s);
                if (lane == 0) s.small[1] = is;
            }
            __syncthreads();
            if (s.small[1]) return;
        }
        // (entries whose weights together do not reach top_p of the row are not sorted)
        bool enough = true;
        if (st.k == 0 && st.tp < 1.0f && complete != 0) {
            double sum;
            before_me(tid < n ? wt((uint32_t)(s.sorted[tid] >> 32)) : 0.0, s.wave, sum);
            enough = sum >= (double)st.tp * total;
        }
        if (enough) {
            sort(s, n, true);
            const unsigned long long e = tid < n ? s.sorted[tid] : 0;
            const uint32_t key = (uint32_t)(e >> 32);
            const bool in = tid < n && (st.k == 0 || tid < st.k);
            const double y = in ? wt(key) : 0.0;
            double sum;
            const double run = before_me(y, s.wave, sum);
            const double goal = (double)st.tp * (st.k > 0 ? sum : total);
            const bool keep = in && (tid == 0 || ((st.tp >= 1.0f || run < goal) && y >= (double)st.low)), sure = tid < n && key >= complete;
            const int kept = __syncthreads_count(keep), certain = __syncthreads_count(sure);
            // the run ends inside what is certain, or with top_k, or with the last entry there is
            done = complete == 0 || !(kept > certain || (kept == certain && kept != st.k) || (st.k > 0 && st.tp < 1.0f && certain < st.k));
            if (done) {
                // what is kept, by index
                double *weights = reinterpret_cast<double *>(s.bins);
                weights[tid] = y;
                __syncthreads();
                if (tid < kept) s.sorted[tid] = ((unsigned long long)(uint32_t)~(uint32_t)e << 32) | (uint32_t)tid;
                sort(s, kept, false);
                const unsigned long long by = tid < kept ? s.sorted[tid] : 0;
                const double v = tid < kept ? weights[(uint32_t)by] : 0.0;
                double kept_sum;
                const double up = before_me(v, s.wave, kept_sum) + v, goal_u = st.u * kept_sum;
                int t = first_of(tid < kept && up > goal_u, s);
                if (t == kEnd) t = last_of(v > 0, s);
                if (tid == t) result(p, r, (int)(by >> 32), v, kept_sum);
                return;
            }
        }
    }
    // ---- read again: what is kept are the entries above `cut`, and of that value those up to index `last`; of weights from low up ----
    float cut = -3.4028234663852886e38f;
    int last = 0x7FFFFFFF;
    int bits = 51;  // of a weight of 1 (whole()), so that the sum of all fits 62
    while ((p.vocab - 1) >> (62 - bits)) bits--;
    const double unit = __longlong_as_double((long long)(1023 + bits) << 52);
    constexpr int AT = 2;  // (four: registers spill, 256 x 128256 with flat rows among them 187 us against 180)
    auto kept_at = [&](float f, int i) { return f > cut || (f == cut && i <= last); };  // (values: NaN is never kept)
    auto each = [&](auto use) {  // use(first of four, values) for every four entries, a wave's stripes one after the other
        for (int b0 = w; b0 < p.stripes; b0 += AT * kWaves) {
            float f[AT][4];
            x.stripes(b0, kWaves, f);
#pragma unroll
            for (int a = 0; a < AT; a++) use((b0 + a * kWaves) * kStripe + 4 * lane, f[a]);
        }
    };
    const double low = (double)st.low;
    auto weigh_at = [&](float f, int i) {
        const double y = wt.of(kept_at(f, i) ? f : __builtin_nanf(""));
        return y >= low ? y : 0.0;
    };
    auto set_mass = [&](int i, double y) { __hip_atomic_store(p.mass + (int64_t)r * p.stripes + i, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto mass_of = [&](int i) { return __hip_atomic_load(p.mass + (int64_t)r * p.stripes + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    // This wave's entries with `is` to s.sorted, as far as there is room; s.small[3] counts them.
    auto collect = [&](int i, const float (&f)[4], const bool (&is)[4]) {
        uint32_t n = 0;
#pragma unroll
        for (int v = 0; v < 4; v++) n += is[v];
        const uint32_t incl = running(n);
        uint32_t base = 0;
        if (lane == 63 && incl != 0) base = atomicAdd(&s.small[3], incl);
        uint32_t at = of_lane(base, 63) + (incl - n);
#pragma unroll
        for (int v = 0; v < 4; v++)
            if (is[v]) {
                if (at < kMost) s.sorted[at] = ((unsigned long long)key_of(f[v]) << 32) | (uint32_t)~(i + v);
                at++;
            }
    };
    // Of the `inside` entries in s.sorted, where those before them weigh `above`: how many the run takes. In order afterwards.
    auto take = [&](int inside, bool weigh, double above, double goal) {
        sort(s, inside, true);
        const unsigned long long e = tid < inside ? s.sorted[tid] : 0;
        const double y = tid < inside ? (weigh ? wt((uint32_t)(e >> 32)) * unit : 1.0) : 0.0;
        double sum;
        const double run = above + before_me(y, s.wave, sum);
        // up to the last entry before which the goal has not been reached
        return last_of(tid < inside && (run < goal || (tid == 0 && above == 0)), s) + 1;
    };
    auto finite = [](uint32_t k) { return k < 0x00800000u ? -3.4028234663852886e38f : of_key(k); };  // the smallest value of key k or above
    for (int phase = 0; phase < 2; phase++) {
        if (phase == 0 ? st.k == 0 : st.tp >= 1.0f) continue;
        const bool weigh = phase == 1;
        double goal = st.k;
        uint32_t lo = 1, hi = top;  // the keys among which the run ends
        double above = 0;           // entries, or weight in units, above them
        double expected = weigh ? st.k : p.vocab;  // entries among them, at least where it is more than can be sorted
        if (weigh && st.k == 0) {   // from the workgroups' bins
            const float per = bins_a_unit(st.t);
            const int first = bin_of(top, per);
            double mine[2] = {};
            static_assert(kBins == 2 * kEnd, "two bins a thread");
            if (tid < p.groups) s.from[tid] = s.weight[tid] > 0 ? (uint32_t)(first - bin_of(lefts[tid].x, per)) : 0;
            __syncthreads();
            constexpr int GA = 8;
            for (int g0 = 0; g0 < p.groups; g0 += GA) {
                unsigned long long a[GA][2];
                double by[GA];
                int off[GA];
#pragma unroll
                for (int v = 0; v < GA; v++) {
                    const int g = g0 + v < p.groups ? g0 + v : g0;
                    by[v] = g0 + v < p.groups ? s.weight[g] * (unit * 0x1p-48) : 0.0;
                    const int at = 2 * tid - (int)s.from[g];
                    const unsigned long long *from = p.hist + ((int64_t)r * p.groups + g) * kBins;
                    off[v] = at;  // (loads without conditions are in flight together)
                    a[v][0] = from[at < 0 ? 0 : at];
                    a[v][1] = from[at < -1 ? 0 : at + 1];
                }
#pragma unroll
                for (int v = 0; v < GA; v++) {
                    mine[0] += off[v] >= 0 ? ldexp((double)a[v][0], -bin_exponent(off[v])) * by[v] : 0.0;
                    mine[1] += off[v] >= -1 ? ldexp((double)a[v][1], -bin_exponent(off[v] + 1)) * by[v] : 0.0;
                }
            }
            goal = (double)st.tp * total * unit;
            double all;
            const double run = before_me(mine[0] + mine[1], s.wave, all);
            const int t = first_of(mine[0] + mine[1] > 0 && run + (mine[0] + mine[1]) >= goal, s);
            __syncthreads();
            if (tid == (t < kEnd ? t : kEnd - 1)) {
                const bool second = t == kEnd || !(mine[0] > 0 && run + mine[0] >= goal);
                s.small[2] = (uint32_t)(2 * tid + second);
                s.sum = t == kEnd ? 0.0 : second ? run + mine[0] : run;
                s.wave[0] = second ? mine[1] : mine[0];
            }
            __syncthreads();
            const int bin = first - (int)s.small[2];
            above = s.sum;
            // the keys of that bin: its number rises with the key
            auto from_bin = [&](int b) {  // the smallest key of bin b or above
                uint32_t a = 1, c = top + 1;
                while (a < c) {
                    const uint32_t mid = a + (c - a) / 2;
                    if (bin_of(mid, per) >= b) c = mid;
                    else a = mid + 1;
                }
                return a;
            };
            if (t < kEnd) {  // (else the run ends below the bins: all keys)
                lo = from_bin(bin);
                hi = from_bin(bin + 1) - 1;
                if (hi < lo) hi = lo;
            }
            expected = t < kEnd ? s.wave[0] / (wt(hi < top ? hi : top) * unit) : p.vocab;
            __syncthreads();
        } else if (weigh) {
            double sum = 0, all;
            each([&](int i, const float (&f)[4]) {
#pragma unroll
                for (int v = 0; v < 4; v++)
                    sum += wt.of(kept_at(f[v], i + v) ? f[v] : __builtin_nanf(""));
            });
            before_me(sum, s.wave, all);
            goal = (double)st.tp * all * unit;
            lo = key_of(cut);
        }
        int inside = 0;
        if (weigh && st.k == 0 && expected <= kMost) {
            // the bin's entries, and at once the stripes' weights above them; if the bin can be sorted, its kept entries are added (1 x 128256,
            // top_p .95: 91 us against 101)
            const float from = finite(lo), to = of_key(hi == 0x7FFFFFFFu ? hi - 1 : hi);
            if (tid == 0) s.small[3] = 0;
            __syncthreads();
            each([&](int i, const float (&f)[4]) {
                bool is[4], some = false;
                double sum = 0;
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    is[v] = f[v] >= from && f[v] <= to, some = some || is[v];
                    const double y = wt.of(f[v] > to ? f[v] : __builtin_nanf(""));
                    sum += y >= low ? y : 0.0;
                }
                sum = wave_sum(sum);
                if (lane == 0 && i < p.vocab) set_mass(i / kStripe, sum);
                if (__any(some)) collect(i, f, is);
            });
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            inside = (int)s.small[3];
            if (inside <= kMost) {
                const int n = take(inside, true, above, goal);
                const unsigned long long e = s.sorted[tid < n ? tid : 0], e_last = s.sorted[n > 0 ? n - 1 : 0];
                cut = n > 0 ? of_key((uint32_t)(e_last >> 32)) : to;
                last = n > 0 ? (int)~(uint32_t)e_last : -1;
                double *weights = reinterpret_cast<double *>(s.bins);
                const double y = tid < n ? wt((uint32_t)(e >> 32)) : 0.0;
                weights[tid] = y >= low ? y : 0.0;
                __syncthreads();
                if (tid < n) s.sorted[tid] = ((unsigned long long)(uint32_t)~(uint32_t)e << 32) | (uint32_t)tid;
                sort(s, n, false);
                auto stripe_of = [&](int i) { return (int)(s.sorted[i] >> 32) / kStripe; };
                if (tid < n && (tid == 0 || stripe_of(tid) != stripe_of(tid - 1))) {
                    double sum = 0;
                    for (int i = tid; i < n && stripe_of(i) == stripe_of(tid); i++) sum += weights[(uint32_t)s.sorted[i]];
                    set_mass(stripe_of(tid), mass_of(stripe_of(tid)) + sum);
                }
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
                return by_stripes(p, r, x, st.u, s, mass_of, [&](uint32_t key, uint32_t i) { return weigh_at(of_key(key), (int)i); });
            }
            __syncthreads();
        }
        // (more than can be sorted, surely: straight to the bins)
        bool many = expected > kMost && lo < hi;
        for (;; many = false) {
            // how many they are, and the first of them
            const float from = finite(lo), to = of_key(hi == 0x7FFFFFFFu ? hi - 1 : hi);  // (that key would be -0, which has 0's)
            if (tid == 0) s.small[3] = many ? kMost + 1 : 0;
            __syncthreads();
            if (!many) each([&](int i, const float (&f)[4]) {
                bool is[4], some = false;
#pragma unroll
                for (int v = 0; v < 4; v++) is[v] = f[v] >= from && f[v] <= to, some = some || is[v];
                if (!__any(some)) return;
#pragma unroll
                for (int v = 0; v < 4; v++) is[v] = is[v] && kept_at(f[v], i + v);
                collect(i, f, is);
            });
            __syncthreads();
            inside = (int)s.small[3];
            if (inside <= kMost || lo == hi) break;
            // too many: in 2048 bins of their keys, from the largest down
            const uint32_t width = (hi - lo) / kBins + 1;
            int *finer = reinterpret_cast<int *>(s.count);  // their units are smaller by the powers of two that their largest weight is below 1
            for (int i = tid; i < kBins; i += kEnd) {
                s.bins[i] = 0;
                if (weigh) {
                    const uint64_t down = (uint64_t)i * width;
                    finer[i] = down < hi ? 1022 - (int)((uint64_t)__double_as_longlong(wt((uint32_t)(hi - down))) >> 52) : 0;
                }
            }
            __syncthreads();
            const float by_width = 1.0f / (float)width;
            auto sub = [&](uint32_t k) {  // (hi - k) / width
                uint32_t q = (uint32_t)((float)(hi - k) * by_width);
                const int64_t rest = (int64_t)(hi - k) - (int64_t)q * width;
                if (rest < 0) q--;
                else if (rest >= (int64_t)width) q++;
                return q < kBins ? q : kBins - 1;
            };
            each([&](int i, const float (&f)[4]) {
#pragma unroll
                for (int v = 0; v < 4; v++)
                    if (f[v] >= from && f[v] <= to && kept_at(f[v], i + v)) {
                        const uint32_t k = key_of(f[v]);
                        const int q = (int)sub(k);
                        atomicAdd(&s.bins[q], weigh ? whole(ldexp(wt(k), bits + finer[q])) : 1ull);
                    }
            });
            __syncthreads();
            const double m0 = ldexp((double)s.bins[2 * tid], weigh ? -finer[2 * tid] : 0), m1 = ldexp((double)s.bins[2 * tid + 1], weigh ? -finer[2 * tid + 1] : 0);
            double all;
            const double run = above + before_me(m0 + m1, s.wave, all);
            int t = first_of(m0 + m1 > 0 && run + (m0 + m1) >= goal, s);
            if (t == kEnd) t = last_of(m0 + m1 > 0, s);  // (a sum that was rounded)
            __syncthreads();
            if (tid == t) {
                const bool second = m1 > 0 && !(m0 > 0 && run + m0 >= goal);
                s.small[2] = (uint32_t)(2 * tid + second);
                s.sum = second ? run + m0 : run;
            }
            __syncthreads();
            above = s.sum;
            const uint32_t q = s.small[2];
            const uint32_t new_hi = hi - q * width;
            lo = new_hi - lo >= width ? new_hi - (width - 1) : lo;
            hi = new_hi;
            __syncthreads();
        }
        if (inside <= kMost) {
            const int n = take(inside, weigh, above, goal);
            const unsigned long long e_last = s.sorted[n > 0 ? n - 1 : 0];
            cut = n > 0 ? of_key((uint32_t)(e_last >> 32)) : of_key(hi);
            last = n > 0 ? (int)~(uint32_t)e_last : -1;  // (none of these: what is above them)
        } else {
            // one key many times: as many as it takes, by index
            double n = weigh ? ceil((goal - above) / (wt(lo) * unit)) : goal - above;
            n = n < 1 ? (above == 0 ? 1 : n) : n;
            const uint32_t take = n < 1 ? 0 : n < (double)inside ? (uint32_t)n : (uint32_t)inside;
            // (a thread's share of the entries, in a row)
            const int per = ((p.vocab + kEnd - 1) / kEnd + 3) & ~3, i0 = tid * per < p.vocab ? tid * per : p.vocab, i1 = i0 + per < p.vocab ? i0 + per : p.vocab;
            uint32_t mine = 0, all;
            for (int i = i0; i < i1; i += 4) {
                float f[4];
                x.values4(i, f);
#pragma unroll
                for (int v = 0; v < 4; v++) mine += f[v] == of_key(lo) && kept_at(f[v], i + v);
            }
            const uint32_t seen = before_me(mine, s.u, all);
            __syncthreads();
            if (take > seen && take <= seen + mine) {
                uint32_t n = seen;
                for (int i = i0; i < i1; i++)
                    if (x.value(i) == of_key(lo) && kept_at(x.value(i), i) && ++n == take) s.small[2] = (uint32_t)i;
            }
            __syncthreads();
            const int at = (int)s.small[2];
            __syncthreads();
            cut = of_key(lo);
            last = take ? at : -1;
        }
        __syncthreads();
    }
    // the stripes' weights
    each([&](int i, const float (&f)[4]) {
        bool some = false;
#pragma unroll
        for (int v = 0; v < 4; v++) some = some || f[v] >= cut;
        double sum = 0;
        if (__any(some)) {
#pragma unroll
            for (int v = 0; v < 4; v++) sum += weigh_at(f[v], i + v);
            sum = wave_sum(sum);
        }
        if (lane == 0 && i < p.vocab) set_mass(i / kStripe, sum);
    });
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    by_stripes(p, r, x, st.u, s, mass_of, [&](uint32_t key, uint32_t i) { return weigh_at(of_key(key), (int)i); });
}

}  // namespace

int launch_sample(trhip_ctx *ctx, const void *logits, int io, int64_t stride, int64_t rows, int64_t vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *u, int *token, float *logprob) {
    const int64_t cus = ctx->sm_count > 0 ? ctx->sm_count : 256, stripes = (vocab + kStripe - 1) / kStripe, esize = io == TRHIP_F32 ? 4 : 2;
    // stripes a wave: few for few rows, so that they lie on many CUs (16 x 151936: twice as many workgroups, four a wave, 14.3 us without a
    // filter, eight 15.7), many for many, whose workgroups' entries and bins are fewer (256 x 128256, top_k 50: eight 45 us, four 48)
    constexpr int WAVES = kRead / 64;
    int64_t each = 1;
    auto groups_of = [&](int64_t j) { return (stripes + WAVES * j - 1) / (WAVES * j); };
    while (each < 8 && rows * groups_of(each) > 2 * cus) each *= 2;
    // (a workgroup's share of a row's largest entries has a part that does not shrink: 1 x 128256 on 63 workgroups leaves too many of k 293
    // to sort, 119 us against 23; on 16 it takes 11.3 without a filter against 10.0)
    while (each < 8 && groups_of(each) > 32) each *= 2;
    const int64_t groups = groups_of(each);  // (at most 1024: one a thread of the second launch)
    const double mean = (double)kMost / 2 / (double)groups;
    int64_t room = (int64_t)(mean + 3.0 * __builtin_sqrt(mean) + 4.0) * 3 / 2 + 16;
    if (room > kMost) room = kMost;
    // rows of a launch: at most 2^28 bytes of workspace where more than one
    const int64_t row_bytes = (stripes + groups * (room + kBins + 2)) * 8;
    int64_t most = ((int64_t)1 << 28) / row_bytes;
    most = most < 1 ? 1 : most > 32768 ? 32768 : most;
    if (most > rows) most = rows;
    int st = TRHIP_OK;
    uint8_t *ws = static_cast<uint8_t *>(workspace(ctx, (size_t)(most * row_bytes), &st));
    if (!ws) return st;
    const int wide = reinterpret_cast<uintptr_t>(logits) % (4 * esize) == 0 && stride % 4 == 0;
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        const int64_t n = rows - r0 < most ? rows - r0 : most;
        SampleArgs p = {static_cast<const char *>(logits) + r0 * stride * esize, io, stride, (int)vocab, (int)stripes, (int)groups, (int)room, wide,
                        temperature ? temperature + r0 : nullptr, top_k ? top_k + r0 : nullptr, top_p ? top_p + r0 : nullptr, min_p ? min_p + r0 : nullptr, u + r0,
                        token + r0, logprob ? logprob + r0 : nullptr, nullptr, nullptr, nullptr, nullptr};
        p.left = reinterpret_cast<uint4 *>(ws);  // (16-byte aligned)
        p.mass = reinterpret_cast<double *>(ws + most * groups * 16);
        p.list = reinterpret_cast<unsigned long long *>(p.mass + most * stripes);
        p.hist = p.list + most * groups * room;
        const dim3 grid((unsigned)groups, (unsigned)n);
        if (each == 1) hipLaunchKernelGGL(sample_read<1>, grid, dim3(kRead), 0, ctx->stream, p);
        else if (each == 2) hipLaunchKernelGGL(sample_read<2>, grid, dim3(kRead), 0, ctx->stream, p);
        else if (each == 4) hipLaunchKernelGGL(sample_read<4>, grid, dim3(kRead), 0, ctx->stream, p);
        else hipLaunchKernelGGL(sample_read<8>, grid, dim3(kRead), 0, ctx->stream, p);
        st = launch_check(ctx, "sample");
        if (st != TRHIP_OK) return st;
        hipLaunchKernelGGL(sample_end, dim3((unsigned)n), dim3(kEnd), 0, ctx->stream, p);
        st = launch_check(ctx, "sample");
        if (st != TRHIP_OK) return st;
    }
    return TRHIP_OK;
}

}  // namespace trhip
