// sample.hip -- the next token of each row of logits: temperature, top-k, top-p and min-p, from a given random number.
//
// One launch that reads every logit once. A row is cut into stripes of 256 entries, dealt in turn to the waves of its workgroups,
// which hold them in registers. A workgroup leaves, as the row's settings need it,
//   the weight of each of its stripes, relative to its own largest logit (rows without a filter, and the sum that top_p is a part of),
//   its largest entries, by a threshold that at least as many of its threads' maxima reach (rows with a filter).
// The row's last workgroup finishes it: without a filter it finds the stripe in which the random number falls, and there the entry;
// with one it sorts the entries that the workgroups left (some hundreds), cuts the run that is kept, and walks it by index. The
// workgroups' shares are what a row whose large entries lie anywhere needs with room to spare; whether they are complete is checked, and a row
// where they are not (a flat one, of which thousands are kept, or one whose largest entries lie in few stripes) goes on to whole(),
// which reads the row again several times.
//
// Weights and their sums are in 64 bits, since one border among a hundred thousand has to be met: e^x by a table of 64 powers and a
// polynomial of degree 5, ten operations.
#include "trhip_internal.hpp"

namespace trhip {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64, kStripe = 256, kMost = 1024;  // kMost: entries that are sorted at most
constexpr int kBins = 2048;

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
    unsigned long long *hist;  // [row][workgroup][kBins]: weight in bins of its logits, from the largest down, in units of 2^-48
    uint32_t *left;         // [row][workgroup][4]: largest key, threshold (0: all entries left), entries left, unused
    uint32_t *arrivals;     // [row]
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
    __device__ __forceinline__ uint32_t key(int i) const {
        return key_of(io == TRHIP_F32 ? static_cast<const float *>(x)[i] : h16_to_f32(static_cast<const uint16_t *>(x)[i], io));
    }
    // entries i .. i + 3 (i a multiple of 4); 0 past the last
    __device__ __forceinline__ void keys4(int i, uint32_t (&k)[4]) const {
        if (wide && i + 4 <= vocab) {
            float f[4];
            if (io == TRHIP_F32) {
                *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
            } else {
                const uint2 y = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(x) + i);
                f[0] = h16_to_f32(y.x & 0xFFFFu, io), f[1] = h16_to_f32(y.x >> 16, io);
                f[2] = h16_to_f32(y.y & 0xFFFFu, io), f[3] = h16_to_f32(y.y >> 16, io);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) k[u] = key_of(f[u]);
        } else {
#pragma unroll
            for (int u = 0; u < 4; u++) k[u] = i + u < vocab ? key(i + u) : 0;
        }
    }
};

// e^((l - max) / T) of a key. e^t = 2^(n / 64) e^r, n = rint(64 t / ln 2), |r| <= ln 2 / 128: what r^6 / 720 leaves out is 2^-54.
struct Weight {
    uint32_t top;
    double max, inv;
    const double *table;  // 2^(j / 64)
    __device__ __forceinline__ double operator()(uint32_t k) const {
        const double t = ((double)of_key(k) - max) * inv;
        if (k == top) return 1.0;
        if (k == 0) return 0.0;
        if (!(t > -700.0)) return exp(t);
        const double n = rint(t * 92.33248261689366);
        const double r = fma(-n, 3.623510646634843e-19, fma(-n, 0.010830424696249145, t));  // (ln 2 / 64 in two parts)
        double y = fma(r, 8.3333333333333332e-3, 4.1666666666666664e-2);
        y = fma(r, y, 1.6666666666666666e-1);
        y = fma(r, y, 0.5);
        y = fma(r, y, 1.0);
        const int i = (int)n;
        const double p = table[i & 63];
        const double s = fma(p, r * y, p);
        return __longlong_as_double(__double_as_longlong(s) + ((long long)(i >> 6) << 52));
    }
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
    s.u = u >= 0.0f ? (double)u : 0.0;
    return s;
}
// How many entries of the whole row its workgroups should cover, and a workgroup's share of them: the mean, four standard deviations of
// entries that lie anywhere, and six.
constexpr int kCover = 256;
__device__ __forceinline__ int share_of(int n, int groups) {
    const float m = (float)n * __builtin_amdgcn_rcpf((float)groups);
    const int s = (int)(m + 4.0f * __builtin_amdgcn_sqrtf(m) + 6.0f);
    return s < n ? s : n;
}

struct Lds {
    double table[64];
    unsigned long long sorted[kMost];
    double weight[kMost];
    union {
        unsigned long long bins[kBins];
        struct {
            uint32_t from[kMost], count[kMost];  // a workgroup's entries
        };
        unsigned long long stripe[kMost];
    };
    uint32_t u[kThreads];
    uint32_t small[16];
    double wave[kWaves];
};

// Bins of a thirty-second of a nat, of logits over the temperature: the number of a key's bin, which rises with it.
__device__ __forceinline__ int bin_of(uint32_t k, float per) {
    return (int)floorf(fminf(fmaxf(of_key(k) * per, -536870912.0f), 536870912.0f));
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
// Over the workgroup; every thread gets the result. (A barrier before the first use of s.u / s.wave is the caller's.)
__device__ uint32_t all_max(uint32_t v, Lds &s) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.u[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s.u[0];
    for (int w = 1; w < kWaves; w++) v = v > s.u[w] ? v : s.u[w];
    return v;
}
__device__ double all_sum(double v, Lds &s) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s.wave[0];
    for (int w = 1; w < kWaves; w++) v += s.wave[w];
    return v;
}
// Sum over the threads before this one, and over all.
template <class T> __device__ T before_me(T v, T *lds, T &total) {
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

// Sorts s.sorted[0 .. n2), n2 a power of two, n2 <= kMost: largest first, or smallest.
__device__ void sort(Lds &s, int n2, bool falling) {
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n2 / 2; i += kThreads) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const unsigned long long x = s.sorted[a], y = s.sorted[b];
                const bool down = ((a & k) == 0) == falling;
                if (down ? x < y : x > y) s.sorted[a] = y, s.sorted[b] = x;
            }
        }
    __syncthreads();
}

__device__ __forceinline__ void result(const SampleArgs &p, int r, int token, double w, double total) {
    p.token[r] = token;
    if (p.logprob) p.logprob[r] = (float)log(w / total);
}

// A row that is kept from `cut` up (of its key the first `ties` by index; weights of at least low): the entry in which u falls.
__device__ void pick(const SampleArgs &p, int r, const Row &x, const Weight &w, uint32_t cut, uint32_t ties, double low, double u, Lds &s) {
    const int tid = threadIdx.x;
    // a thread's share: whole fours, in a row
    const int each = ((p.vocab + kThreads - 1) / kThreads + 3) & ~3, i0 = tid * each < p.vocab ? tid * each : p.vocab, i1 = i0 + each < p.vocab ? i0 + each : p.vocab;
    uint32_t eq = 0, total_eq, eq0 = 0;
    if (ties != 0xFFFFFFFFu) {
        for (int i = i0; i < i1; i += 4) {
            uint32_t k[4];
            x.keys4(i, k);
            for (int v = 0; v < 4; v++) eq += k[v] == cut;
        }
        eq0 = before_me(eq, s.u, total_eq);
    }
    auto walk = [&](auto use) {
        uint32_t n = eq0;
        for (int i = i0; i < i1; i += 4) {
            uint32_t k[4];
            x.keys4(i, k);
            for (int v = 0; v < 4; v++) {
                const bool keep = k[v] != 0 && (k[v] > cut || (k[v] == cut && n < ties));
                n += k[v] == cut;
                if (!keep) continue;
                const double y = w(k[v]);
                if (y >= low) use(i + v, y);
            }
        }
    };
    double sum = 0, total;
    walk([&](int, double y) { sum += y; });
    const double start = before_me(sum, s.wave, total), goal = u * total;
    __syncthreads();
    if (tid == 0) s.small[0] = 0x7FFFFFFF, s.small[1] = 0;
    __syncthreads();
    uint32_t found = 0x7FFFFFFF, last = 0;
    double run = start;
    if (sum > 0)
        walk([&](int i, double y) {
            run += y;
            if (y > 0) last = (uint32_t)i;
            if (run > goal && found == 0x7FFFFFFF) found = (uint32_t)i;
        });
    if (found != 0x7FFFFFFF) atomicMin(&s.small[0], found);
    if (last) atomicMax(&s.small[1], last);
    __syncthreads();
    if (tid == 0) {
        const int token = (int)(s.small[0] != 0x7FFFFFFF ? s.small[0] : s.small[1]);
        result(p, r, token, w(x.key(token)), total);
    }
}

__device__ __forceinline__ uint32_t agent_get(const uint32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned long long agent_get(const unsigned long long *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ double agent_get(const double *p) {
    return __longlong_as_double((long long)agent_get(reinterpret_cast<const unsigned long long *>(p)));
}
template <class T> __device__ __forceinline__ void agent_put(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The entry of stripe `at` (keys k, four a lane) in which the goal falls, the weights before the stripe being `before`; by one wave.
template <class F>
__device__ __forceinline__ void last_stripe(const SampleArgs &p, int r, int at, double before, double goal, double total, const uint32_t (&k)[4], F weight) {
    const int lane = threadIdx.x & 63;
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
    const int src = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
    if (lane == src) result(p, r, at * kStripe + 4 * lane + (over ? found : last), over ? chosen : final, total);
}

// Sorts one element a lane: largest first, or smallest.
__device__ __forceinline__ unsigned long long sort64(unsigned long long e, bool falling) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            const unsigned long long o = __shfl_xor(e, j);
            const bool first = (lane & j) == 0, down = ((lane & k) == 0) == falling;  // this lane keeps the larger one
            e = (first == down) == (e > o) ? e : o;
        }
    return e;
}

// A filtered row whose kept run is among its largest 64 entries, by one wave: those that a threshold leaves of the n in s.sorted.
// False: it is not, or that is not certain.
__device__ bool top64(const SampleArgs &p, int r, const Weight &wt, const Setting &st, double total, uint32_t complete, int n, Lds &s) {
    const int lane = threadIdx.x & 63;
    constexpr int PER = kMost / 64;
    uint32_t k[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) k[i] = 64 * i + lane < n ? (uint32_t)(s.sorted[64 * i + lane] >> 32) : 0;
    uint32_t lo = 1, hi = wt.top;  // at least `want` entries reach lo
    int count = n;
    const int want = st.k > 0 ? st.k : 48;
    for (int step = 0; step < 40 && count > 64 && lo < hi; step++) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) c += __popcll(__ballot(k[i] >= mid));
        if (c >= want) lo = mid, count = c;
        else hi = mid - 1;
    }
    if (count > 64) return false;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const uint64_t m = __ballot(k[i] >= lo);
        if (k[i] >= lo) s.weight[at + __popcll(m & (((uint64_t)1 << lane) - 1))] = __longlong_as_double((long long)s.sorted[64 * i + lane]);
        at += __popcll(m);
    }
    __builtin_amdgcn_wave_barrier();
    unsigned long long e = lane < count ? (unsigned long long)__double_as_longlong(s.weight[lane]) : 0;
    e = sort64(e, true);
    const uint32_t key = (uint32_t)(e >> 32);
    const bool in = lane < count && (st.k == 0 || lane < st.k);
    const double w = in ? wt(key) : 0.0, incl = running(w), before = before_lane(incl), sum = of_lane(incl, 63);
    // every entry from here up is in these lanes
    const uint32_t from = count < n && lo > complete ? lo : complete;
    const bool sure = lane < count && key >= from, all = from == 0 || (from <= 1 && complete == 0);
    const double goal = (double)st.tp * (st.k > 0 ? sum : total);
    const bool keep = in && (lane == 0 || ((st.tp >= 1.0f || before < goal) && w >= (double)st.low));
    const int kept = __popcll(__ballot(keep)), certain = __popcll(__ballot(sure));
    if (!all) {
        if (kept > certain || (kept == certain && kept != st.k)) return false;  // (the run may go on past what is here)
        if (st.k > 0 && st.tp < 1.0f && certain < st.k) return false;           // (nor is the sum certain)
    }
    unsigned long long by = keep ? ((unsigned long long)(uint32_t)~(uint32_t)e << 32) | (uint32_t)lane : ~0ull;
    by = sort64(by, false);
    const double v = __shfl(w, (int)((uint32_t)by & 63)), mine = lane < kept ? v : 0.0, run = running(mine), kept_sum = of_lane(run, 63), goal_u = st.u * kept_sum;
    const uint64_t over = __ballot(lane < kept && run > goal_u), some = __ballot(lane < kept && v > 0);
    const int pos = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
    const uint32_t token = of_lane((uint32_t)(by >> 32), pos);
    const double chosen = of_lane(mine, pos);
    if (lane == 0) result(p, r, (int)token, chosen, kept_sum);
    return true;
}

// A row without top_k whose kept run is long: the bin in which it ends, from the workgroups' bins; then one pass over the row, which weighs the
// stripes' entries above that bin and takes the bin's own entries out to sort them; then the stripe in which u falls.
__device__ __noinline__ void sweep(const SampleArgs &p, int r, const Row &x, const Weight &wt, const Setting &st, double total, Lds &s);
__device__ __noinline__ void whole(const SampleArgs &p, int r, const Row &x, const Weight &w, const Setting &st, Lds &s);

__device__ __noinline__ void sweep(const SampleArgs &p, int r, const Row &x, const Weight &wt, const Setting &st, double total, Lds &s) {
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float per = 32.0f / st.t;
    const int first = bin_of(wt.top, per);
    const double low = (double)st.low, goal = (double)st.tp * total;
    int end = 0x7FFFFFFF;  // the bin in which the run ends, counted from the largest logit's down
    double above = 0;      // the weight of those before it
    if (st.tp < 1.0f) {
        static_assert(kBins == 4 * kThreads, "four bins a thread");
        double mine[4] = {};
        const uint32_t *lefts = p.left + (int64_t)r * p.groups * 4;
        for (int g = 0; g < p.groups; g++) {
            const uint32_t a = agent_get(lefts + 4 * g);
            if (a == 0) continue;
            const int shift = first - bin_of(a, per);
            const double unit = wt(a) * 0x1p-48;
            const unsigned long long *from = p.hist + ((int64_t)r * p.groups + g) * kBins;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = 4 * tid + i - shift;
                if (at >= 0) mine[i] += (double)agent_get(from + at) * unit;
            }
        }
        double all;
        double run = before_me((mine[0] + mine[1]) + (mine[2] + mine[3]), s.wave, all);
        __syncthreads();
        if (tid == 0) s.small[5] = kBins - 1;
        __syncthreads();
        const double start = run;
        for (int i = 0; i < 4; i++) {
            run += mine[i];
            if (mine[i] > 0 && run >= goal) {
                atomicMin(&s.small[5], (uint32_t)(4 * tid + i));
                break;
            }
        }
        __syncthreads();
        end = (int)s.small[5];
        if (end >> 2 == tid) {
            run = start;
            for (int i = 0; i < (end & 3); i++) run += mine[i];
            s.wave[0] = run;
        }
        __syncthreads();
        above = s.wave[0];
        __syncthreads();
    }
    // the stripes' weights, in units of 2^-44, and the entries of the last bin
    if (tid == 0) s.small[6] = 0;
    for (int i = tid; i < kMost; i += kThreads) s.stripe[i] = 0;
    __syncthreads();
    constexpr int AT = 4;
    for (int b0 = w; b0 < p.stripes; b0 += AT * kWaves) {
        uint32_t k[AT][4];
#pragma unroll
        for (int a = 0; a < AT; a++) {
            if (b0 + a * kWaves < p.stripes) x.keys4((b0 + a * kWaves) * kStripe + 4 * lane, k[a]);
            else k[a][0] = k[a][1] = k[a][2] = k[a][3] = 0;
        }
#pragma unroll
        for (int a = 0; a < AT; a++) {
            double sum = 0;
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int b = k[a][v] ? first - bin_of(k[a][v], per) : 0x7FFFFFFF;
                const bool in = k[a][v] != 0 && b < end, is = k[a][v] != 0 && b == end;
                if (__any(in)) {
                    const double y = in ? wt(k[a][v]) : 0.0;
                    sum += y >= low ? y : 0.0;
                }
                const uint64_t m = __ballot(is);
                if (m) {
                    uint32_t at = 0;
                    if (lane == 0) at = atomicAdd(&s.small[6], (uint32_t)__popcll(m));
                    at = __builtin_amdgcn_readfirstlane(at) + __popcll(m & (((uint64_t)1 << lane) - 1));
                    if (is && at < kMost) s.sorted[at] = ((unsigned long long)k[a][v] << 32) | (uint32_t)~((b0 + a * kWaves) * kStripe + 4 * lane + v);
                }
            }
            const double all = wave_sum(sum);
            if (lane == 0 && b0 + a * kWaves < p.stripes) s.stripe[b0 + a * kWaves] = (unsigned long long)rint(all * 0x1p44);
        }
    }
    __syncthreads();
    const int n = (int)s.small[6];
    if (n > kMost) return whole(p, r, x, wt, st, s);
    unsigned long long least = ~0ull;  // the last entry that is kept of that bin
    if (n > 0) {
        int n2 = 2;
        while (n2 < n) n2 <<= 1;
        for (int i = n + tid; i < n2; i += kThreads) s.sorted[i] = 0;
        sort(s, n2, true);
        const unsigned long long e0 = 2 * tid < n ? s.sorted[2 * tid] : 0, e1 = 2 * tid + 1 < n ? s.sorted[2 * tid + 1] : 0;
        const double w0 = e0 ? wt((uint32_t)(e0 >> 32)) : 0.0, w1 = e1 ? wt((uint32_t)(e1 >> 32)) : 0.0;
        double sum;
        const double run0 = above + before_me(w0 + w1, s.wave, sum), run1 = run0 + w0;
        const bool keep0 = e0 && ((end == 0 && tid == 0) || (run0 < goal && w0 >= low)), keep1 = e1 && run1 < goal && w1 >= low;
        if (keep0) atomicAdd(&s.stripe[(uint32_t)~(uint32_t)e0 / kStripe], (unsigned long long)rint(w0 * 0x1p44));
        if (keep1) atomicAdd(&s.stripe[(uint32_t)~(uint32_t)e1 / kStripe], (unsigned long long)rint(w1 * 0x1p44));
        const int kept = __syncthreads_count(keep0) + __syncthreads_count(keep1);
        if (kept > 0) least = s.sorted[kept - 1];
    }
    __syncthreads();
    static_assert(kMost == 2 * kThreads, "two stripes a thread");
    const double m0 = (double)s.stripe[2 * tid] * 0x1p-44, m1 = (double)s.stripe[2 * tid + 1] * 0x1p-44;
    double kept_sum;
    const double before = before_me(m0 + m1, s.wave, kept_sum), goal_u = st.u * kept_sum;
    __syncthreads();
    if (tid == 0) s.small[2] = 0x7FFFFFFF, s.small[3] = 0;
    __syncthreads();
    if (m0 > 0 && before + m0 > goal_u) atomicMin(&s.small[2], (uint32_t)(2 * tid));
    if (m1 > 0 && before + m0 + m1 > goal_u) atomicMin(&s.small[2], (uint32_t)(2 * tid + 1));
    if (m0 > 0) atomicMax(&s.small[3], (uint32_t)(2 * tid));
    if (m1 > 0) atomicMax(&s.small[3], (uint32_t)(2 * tid + 1));
    __syncthreads();
    const int at = (int)(s.small[2] != 0x7FFFFFFF ? s.small[2] : s.small[3]);
    if (at >> 1 == tid) s.wave[0] = at & 1 ? before + m0 : before;
    __syncthreads();
    if (w == 0) {
        uint32_t k[4];
        x.keys4(at * kStripe + 4 * lane, k);
        auto weight = [&](uint32_t key, uint32_t i) {
            if (key == 0) return 0.0;
            const int b = first - bin_of(key, per);
            if (b > end || (b == end && ((((unsigned long long)key << 32) | (uint32_t)~i) < least || least == ~0ull))) return 0.0;
            const double y = wt(key);
            return y >= low || key == wt.top ? y : 0.0;
        };
        last_stripe(p, r, at, s.wave[0], goal_u, kept_sum, k, weight);
    }
}

// A row by itself: the cut by top-k, then by top-p, each by counting (or weighing) entries in bins of the key, eight bits at a time
// from the top.
__device__ __noinline__ void whole(const SampleArgs &p, int r, const Row &x, const Weight &w, const Setting &st, Lds &s) {
    const int tid = threadIdx.x;
    uint32_t cut = 1, ties = 0xFFFFFFFFu;  // kept: keys above cut, and the first `ties` of cut
    int bits = 62;
    while ((p.vocab - 1) >> (62 - bits)) bits--;
    const double unit = __longlong_as_double((long long)(1023 + bits) << 52);
    const int fours = (p.vocab + 3) / 4;
    auto each = [&](auto use) {
        for (int i = tid; i < fours; i += kThreads) {
            uint32_t k[4];
            x.keys4(4 * i, k);
            for (int v = 0; v < 4; v++) use(k[v]);
        }
    };
    for (int phase = 0; phase < 2; phase++) {
        double goal;  // entries, or weight, to reach
        if (phase == 0) {
            if (st.k == 0) continue;
            goal = st.k;
        } else {
            if (!(st.tp < 1.0f)) continue;
            double sum = 0;
            each([&](uint32_t k) {
                if (k > cut || (k == cut && ties == 0xFFFFFFFFu)) sum += w(k);
            });
            sum = all_sum(sum, s);
            if (ties != 0xFFFFFFFFu) sum += (double)ties * w(cut);
            goal = (double)st.tp * sum * unit;
        }
        uint32_t prefix = 0, mask = 0;
        unsigned long long above = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) s.bins[tid] = 0;
            __syncthreads();
            each([&](uint32_t k) {
                if ((k & mask) != prefix || k < cut) return;
                if (phase == 0) atomicAdd(&s.bins[k >> shift & 255], 1ull);
                else if (k > cut || ties == 0xFFFFFFFFu) atomicAdd(&s.bins[k >> shift & 255], (unsigned long long)rint(w(k) * unit));
            });
            __syncthreads();
            if (tid == 0) {
                if (phase == 1 && ties != 0xFFFFFFFFu && (cut & mask) == prefix) s.bins[cut >> shift & 255] += (unsigned long long)(rint(w(cut) * unit) * ties);
                unsigned long long run = above;
                int at = -1;
                for (int b = 255; b >= 0; b--) {
                    const unsigned long long n = s.bins[b];
                    if (n == 0) continue;
                    at = b;
                    above = run;
                    run += n;
                    if ((double)run >= goal) break;
                }
                s.small[0] = at < 0 ? 0 : at;
                s.bins[256] = above;
            }
            __syncthreads();
            above = s.bins[256];
            prefix |= s.small[0] << shift;
            mask |= 255u << shift;
        }
        // of key `prefix` as many as it takes
        if (phase == 0) {
            ties = (uint32_t)(st.k - (int)above);
        } else {
            double n = ceil((goal - (double)above) / rint(w(prefix) * unit));
            n = n < 1 ? 1 : n;
            const uint32_t most = prefix == cut ? ties : 0xFFFFFFFFu;
            ties = n < (double)most ? (uint32_t)n : most;
        }
        cut = prefix;
        __syncthreads();
    }
    pick(p, r, x, w, cut, ties, (double)st.low, st.u, s);
}

template <int J> __global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs p) {
    __shared__ Lds s;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r = blockIdx.y, g = blockIdx.x;
    const Row x = {static_cast<const char *>(p.logits) + r * p.stride * (p.io == TRHIP_F32 ? 4 : 2), p.io, p.vocab, p.wide};
    const Setting st = setting_of(p, r);
    const bool filtered = st.k > 0 || st.tp < 1.0f || st.low > 0.0f, weigh = !filtered || (st.k == 0 && st.tp < 1.0f);
    uint32_t key[J][4], top = 0;
    auto stripe = [&](int j) { return g + p.groups * (w + kWaves * j); };
#pragma unroll
    for (int j = 0; j < J; j++) {
        if (stripe(j) < p.stripes) x.keys4(stripe(j) * kStripe + 4 * lane, key[j]);
        else key[j][0] = key[j][1] = key[j][2] = key[j][3] = 0;
    }
    if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int v = 0; v < 4; v++) top = top > key[j][v] ? top : key[j][v];
    s.u[tid] = top;
    if (tid == 0) s.small[0] = 0;
    __syncthreads();
    uint32_t mine[kWaves];  // every wave has all threads' maxima
    top = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        mine[i] = s.u[64 * i + lane];
        top = top > mine[i] ? top : mine[i];
    }
    top = wave_max(top);
    if (weigh && top != 0) {
        const Weight wt = {top, (double)of_key(top), st.greedy ? 1.0 : 1.0 / (double)st.t, s.table};
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (stripe(j) >= p.stripes) break;
            const double sum = wave_sum((wt(key[j][0]) + wt(key[j][1])) + (wt(key[j][2]) + wt(key[j][3])));
            if (lane == 0) agent_put(p.mass + (int64_t)r * p.stripes + stripe(j), sum);
        }
    }
    if (st.k == 0 && st.tp < 1.0f && top != 0) {
        for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
        __syncthreads();
        const Weight wt = {top, (double)of_key(top), 1.0 / (double)st.t, s.table};
        const float per = 32.0f / st.t;
        const int first = bin_of(top, per);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                if (key[j][v] == 0) continue;
                const int b = first - bin_of(key[j][v], per);
                atomicAdd(&s.bins[b < kBins ? b : kBins - 1], (unsigned long long)rint(wt(key[j][v]) * 0x1p48));
            }
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads) agent_put(p.hist + ((int64_t)r * p.groups + g) * kBins + i, s.bins[i]);
    }
    uint32_t bound = 0, left = 0;
    if (filtered && top != 0) {
        const int cover = st.k > 0 ? st.k : kCover;
        const int share = share_of(cover, p.groups);
        const bool many = share * 11 / 10 * p.groups > kMost || share * 5 / 4 + 8 > p.room;  // (too many to sort)
        if (many) {
            left = 0xFFFFFFFFu;
        } else {
            // a threshold that `share` to share * 9 / 8 threads' maxima reach: halving between the smallest and the largest
            uint32_t lo = 0, hi = top;  // count(>= lo) >= share (or lo is 0)
            bound = 0;
            for (int step = 0; step < 32 && lo < hi; step++) {
                const uint32_t mid = step == 0 ? top : lo + (hi - lo + 1) / 2;
                int n = 0;
#pragma unroll
                for (int i = 0; i < kWaves; i++) n += __popcll(__ballot(mine[i] >= mid));
                if (n >= share) {
                    lo = mid;
                    if (n <= share + share / 8) break;
                } else {
                    hi = mid - 1;
                }
            }
            bound = lo;
            unsigned long long *to = p.list + ((int64_t)r * p.groups + g) * p.room;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const bool is = key[j][v] != 0 && key[j][v] >= bound;
                    const uint64_t m = __ballot(is);
                    if (m == 0) continue;
                    uint32_t at = 0;
                    if (lane == 0) at = atomicAdd(&s.small[0], (uint32_t)__popcll(m));
                    at = __builtin_amdgcn_readfirstlane(at) + __popcll(m & (((uint64_t)1 << lane) - 1));
                    if (is && at < (uint32_t)p.room)
                        agent_put(to + at, ((unsigned long long)key[j][v] << 32) | (uint32_t)~(stripe(j) * kStripe + 4 * lane + v));
                }
            __syncthreads();
            left = s.small[0];
        }
    }
    if (tid == 0) {
        uint32_t *mine_left = p.left + ((int64_t)r * p.groups + g) * 4;
        agent_put(mine_left, top);
        agent_put(mine_left + 1, bound);
        agent_put(mine_left + 2, left);
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);  // this thread's stores have completed
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (tid == 0) {
        const bool last = __hip_atomic_fetch_add(&p.arrivals[r], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)p.groups - 1;
        if (last) agent_put(&p.arrivals[r], 0u);
        s.small[1] = last;
    }
    __syncthreads();
    if (!s.small[1]) return;

    // ---- the row's last workgroup ----
    const uint32_t *lefts = p.left + (int64_t)r * p.groups * 4;
    uint32_t row_top = 0, complete = 0, total_left = 0;
    for (int i = tid; i < p.groups; i += kThreads) {
        const uint32_t a = agent_get(lefts + 4 * i), b = agent_get(lefts + 4 * i + 1), n = agent_get(lefts + 4 * i + 2);
        row_top = row_top > a ? row_top : a;
        complete = complete > b ? complete : b;  // every entry from here up has been left by its workgroup
        total_left = n > (uint32_t)p.room || total_left > kMost ? 0x7FFFFFFFu : total_left + n;
    }
    row_top = all_max(row_top, s);
    if (row_top == 0) {
        if (tid == 0) {
            p.token[r] = -1;
            if (p.logprob) p.logprob[r] = __builtin_nanf("");
        }
        return;
    }
    const Weight wt = {row_top, (double)of_key(row_top), st.greedy ? 1.0 : 1.0 / (double)st.t, s.table};
    // the stripes' weights, relative to the row's largest logit: a thread's share of the stripes in a row
    double total = 0, before = 0;
    const int each = (p.stripes + kThreads - 1) / kThreads, s0 = tid * each < p.stripes ? tid * each : p.stripes, s1 = s0 + each < p.stripes ? s0 + each : p.stripes;
    auto stripe_mass = [&](int i) {
        const uint32_t a = agent_get(lefts + 4 * (i % p.groups));
        return a == 0 ? 0.0 : agent_get(p.mass + (int64_t)r * p.stripes + i) * wt(a);
    };
    if (weigh) {
        double sum = 0;
        for (int i = s0; i < s1; i++) sum += stripe_mass(i);
        before = before_me(sum, s.wave, total);
    }
    if (!filtered) {
        const double goal = st.u * total;
        __syncthreads();
        if (tid == 0) s.small[2] = 0x7FFFFFFF, s.small[3] = 0;
        __syncthreads();
        double run = before;
        for (int i = s0; i < s1; i++) {
            const double y = stripe_mass(i);
            if (y > 0) atomicMax(&s.small[3], (uint32_t)i);
            if (run + y > goal && y > 0) {
                atomicMin(&s.small[2], (uint32_t)i);
                break;
            }
            run += y;
        }
        __syncthreads();
        const int at = (int)(s.small[2] != 0x7FFFFFFF ? s.small[2] : s.small[3]);  // (none: u of 1 and above)
        if (at >= s0 && at < s1) {
            run = before;
            for (int i = s0; i < at; i++) run += stripe_mass(i);
            s.wave[0] = run;
        }
        __syncthreads();
        if (w != 0) return;
        uint32_t k[4];
        x.keys4(at * kStripe + 4 * lane, k);
        last_stripe(p, r, at, s.wave[0], goal, total, k, [&](uint32_t key, uint32_t) { return wt(key); });
        return;
    }
    complete = all_max(complete, s);
    uint32_t n_all;
    const uint32_t n_before = before_me(total_left, s.u, n_all);
    const uint32_t worst = all_max(total_left, s);
    const double goal_all = (double)st.tp * total;
    auto otherwise = [&] {
        // (sweep's sums end at 2^-45 of the largest weight: smaller ones are kept by the smallest min_p alone)
        if (st.k == 0 && p.stripes <= kMost && (st.tp < 1.0f || st.low > 0x1p-40f)) sweep(p, r, x, wt, st, total, s);
        else whole(p, r, x, wt, st, s);
    };
    if (worst > kMost || n_all > kMost) return otherwise();
    {
        uint32_t from = n_before;
        for (int i = tid; i < p.groups; i += kThreads) {
            const uint32_t n = agent_get(lefts + 4 * i + 2);
            s.from[i] = from, s.count[i] = n;
            from += n;
        }
        __syncthreads();
        constexpr int AT = 4;
        for (int i0 = tid; i0 < p.groups * p.room; i0 += AT * kThreads) {
            unsigned long long e[AT];
            uint32_t to[AT];
#pragma unroll
            for (int v = 0; v < AT; v++) {
                const int i = i0 + v * kThreads, gi = i < p.groups * p.room ? i / p.room : 0, slot = i - gi * p.room;
                const bool is = i < p.groups * p.room && (uint32_t)slot < s.count[gi];
                to[v] = is ? s.from[gi] + slot : 0xFFFFFFFFu;
                e[v] = is ? agent_get(p.list + ((int64_t)r * p.groups + gi) * p.room + slot) : 0;
            }
#pragma unroll
            for (int v = 0; v < AT; v++)
                if (to[v] != 0xFFFFFFFFu) s.sorted[to[v]] = e[v];
        }
        __syncthreads();
    }
    if (st.k <= 64) {
        if (w == 0) {
            const bool done = top64(p, r, wt, st, total, complete, (int)n_all, s);
            if (lane == 0) s.small[4] = done;
        }
        __syncthreads();
        if (s.small[4]) return;
    }
    int n = (int)n_all, n2 = 2;
    while (n2 < n) n2 <<= 1;
    for (int i = n + tid; i < n2; i += kThreads) s.sorted[i] = 0;
    sort(s, n2, true);
    // weights and their running sum, two entries a thread
    static_assert(kMost == 2 * kThreads, "two entries a thread");
    const uint32_t k0 = (uint32_t)(s.sorted[2 * tid < n2 ? 2 * tid : 0] >> 32), k1 = (uint32_t)(s.sorted[2 * tid + 1 < n2 ? 2 * tid + 1 : 0] >> 32);
    const bool in0 = 2 * tid < n && (st.k == 0 || 2 * tid < st.k), in1 = 2 * tid + 1 < n && (st.k == 0 || 2 * tid + 1 < st.k);
    const double w0 = in0 ? wt(k0) : 0.0, w1 = in1 ? wt(k1) : 0.0;
    double sum;
    const double run0 = before_me(w0 + w1, s.wave, sum), run1 = run0 + w0;
    // entries that are certain: all of those from `complete` up are here
    const bool sure0 = 2 * tid < n && k0 >= complete, sure1 = 2 * tid + 1 < n && k1 >= complete;
    const double goal = st.k > 0 ? (double)st.tp * sum : goal_all;
    const bool keep0 = in0 && (tid == 0 || ((st.tp >= 1.0f || run0 < goal) && w0 >= (double)st.low));
    const bool keep1 = in1 && (st.tp >= 1.0f || run1 < goal) && w1 >= (double)st.low;
    const int kept = __syncthreads_count(keep0) + __syncthreads_count(keep1);
    const bool doubt = (keep0 && !sure0) || (keep1 && !sure1);
    // (the run ends inside what is certain, or with top_k, or with the last entry there is)
    const bool end = complete == 0 || (st.k > 0 && kept == st.k);
    const int sure = __syncthreads_count(sure0) + __syncthreads_count(sure1);
    if (__syncthreads_or(doubt) || (!end && kept >= sure) || (st.k > 0 && st.tp < 1.0f && sure < (st.k < n ? st.k : n) && complete != 0) || (st.k > n && complete != 0))
        return otherwise();
    // what is kept, by index
    unsigned long long e0 = 0, e1 = 0;
    if (2 * tid < n2) e0 = s.sorted[2 * tid], e1 = s.sorted[2 * tid + 1];
    s.weight[2 * tid] = w0, s.weight[2 * tid + 1] = w1;
    n2 = 2;
    while (n2 < kept) n2 <<= 1;
    __syncthreads();
    const unsigned long long none = ~0ull;
    if (2 * tid < n2) s.sorted[2 * tid] = keep0 ? ((unsigned long long)(uint32_t)~(uint32_t)e0 << 32) | (uint32_t)(2 * tid) : none;
    if (2 * tid + 1 < n2) s.sorted[2 * tid + 1] = keep1 ? ((unsigned long long)(uint32_t)~(uint32_t)e1 << 32) | (uint32_t)(2 * tid + 1) : none;
    sort(s, n2, false);
    const bool a0 = 2 * tid < kept, a1 = 2 * tid + 1 < kept;
    const double v0 = a0 ? s.weight[(uint32_t)s.sorted[2 * tid]] : 0.0, v1 = a1 ? s.weight[(uint32_t)s.sorted[2 * tid + 1]] : 0.0;
    double kept_sum;
    const double q0 = before_me(v0 + v1, s.wave, kept_sum) + v0, q1 = q0 + v1, at = st.u * kept_sum;
    __syncthreads();
    if (tid == 0) s.small[2] = 0x7FFFFFFF, s.small[3] = 0;
    __syncthreads();
    if (a0 && q0 > at) atomicMin(&s.small[2], (uint32_t)(2 * tid));
    if (a1 && q1 > at) atomicMin(&s.small[2], (uint32_t)(2 * tid + 1));
    if (a0 && v0 > 0) atomicMax(&s.small[3], (uint32_t)(2 * tid));
    if (a1 && v1 > 0) atomicMax(&s.small[3], (uint32_t)(2 * tid + 1));
    __syncthreads();
    if (tid == 0) {
        const unsigned long long e = s.sorted[s.small[2] != 0x7FFFFFFF ? s.small[2] : s.small[3]];
        result(p, r, (int)(e >> 32), s.weight[(uint32_t)e], kept_sum);
    }
}

}  // namespace

int launch_sample(trhip_ctx *ctx, const void *logits, int io, int64_t stride, int64_t rows, int64_t vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *u, int *token, float *logprob) {
    const int64_t cus = ctx->sm_count > 0 ? ctx->sm_count : 256, stripes = (vocab + kStripe - 1) / kStripe, esize = io == TRHIP_F32 ? 4 : 2;
    // stripes a wave: few for few rows, so that they lie on many CUs
    int64_t each = 1;
    auto groups_of = [&](int64_t j) { return (stripes + kWaves * j - 1) / (kWaves * j); };
    while (each < 8 && rows * groups_of(each) > 2 * cus) each *= 2;
    while (each < 8 && groups_of(each) > kThreads / 8) each *= 2;
    const int64_t groups = groups_of(each);
    const double mean = (double)kMost / 2 / (double)groups;
    int64_t room = (int64_t)(mean + 4.0 * __builtin_sqrt(mean) + 6.0) * 3 / 2 + 16;
    if (room > kMost) room = kMost;
    // rows of a launch: an arrival counter each, and at most 2^28 bytes of workspace where more than one row
    const int64_t row_bytes = (stripes + groups * (room + kBins + 2)) * 8;
    int64_t most = (int64_t)1 << 28;
    most = most / row_bytes < 1 ? 1 : most / row_bytes;
    if (most > 32768) most = 32768;
    if (most > rows) most = rows;
    int st = TRHIP_OK;
    uint8_t *ws = static_cast<uint8_t *>(workspace(ctx, (size_t)(most * row_bytes), &st));
    if (!ws) return st;
    const int wide = reinterpret_cast<uintptr_t>(logits) % (4 * esize) == 0 && stride % 4 == 0;
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        const int64_t n = rows - r0 < most ? rows - r0 : most;
        SampleArgs p = {static_cast<const char *>(logits) + r0 * stride * esize, io, stride, (int)vocab, (int)stripes, (int)groups, (int)room, wide,
                        temperature ? temperature + r0 : nullptr, top_k ? top_k + r0 : nullptr, top_p ? top_p + r0 : nullptr, min_p ? min_p + r0 : nullptr, u + r0,
                        token + r0, logprob ? logprob + r0 : nullptr, reinterpret_cast<double *>(ws),
                        reinterpret_cast<unsigned long long *>(ws + most * stripes * 8), reinterpret_cast<unsigned long long *>(ws + most * (stripes + groups * room) * 8),
                        reinterpret_cast<uint32_t *>(ws + most * (stripes + groups * (room + kBins)) * 8), ctx->arrivals};
        const dim3 grid((unsigned)groups, (unsigned)n);
        if (each == 1) hipLaunchKernelGGL(sample_kernel<1>, grid, dim3(kThreads), 0, ctx->stream, p);
        else if (each == 2) hipLaunchKernelGGL(sample_kernel<2>, grid, dim3(kThreads), 0, ctx->stream, p);
        else if (each == 4) hipLaunchKernelGGL(sample_kernel<4>, grid, dim3(kThreads), 0, ctx->stream, p);
        else hipLaunchKernelGGL(sample_kernel<8>, grid, dim3(kThreads), 0, ctx->stream, p);
        st = launch_check(ctx, "sample");
        if (st != TRHIP_OK) return st;
    }
    return TRHIP_OK;
}

}  // namespace trhip
