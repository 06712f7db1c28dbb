// sample.hip -- the next token of each row of logits: temperature, top-k, top-p and min-p, from a given random number.
#include "trhip_internal.hpp"

namespace trhip {
namespace {

struct SampleArgs {
    const void *logits;
    int io;
    int64_t stride;
    int vocab;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    int *token;
    float *logprob;
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;

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
    int io, vocab;
    __device__ __forceinline__ uint32_t key(int i) const {
        return key_of(io == TRHIP_F32 ? static_cast<const float *>(x)[i] : h16_to_f32(static_cast<const uint16_t *>(x)[i], io));
    }
};
struct Weight {
    uint32_t top;
    double max, inv;
    __device__ __forceinline__ double operator()(uint32_t k) const {
        return k == top ? 1.0 : k == 0 ? 0.0 : exp(((double)of_key(k) - max) * inv);
    }
};

template <class T> __device__ T sum_all(T v, T *lds) {
    const int tid = threadIdx.x;
    lds[tid] = v;
    __syncthreads();
    for (int o = kThreads / 2; o; o >>= 1) {
        if (tid < o) lds[tid] += lds[tid + o];
        __syncthreads();
    }
    v = lds[0];
    __syncthreads();
    return v;
}
template <class T> __device__ T before_me(T v, T *lds, T &total) {  // sum over the threads before this one
    const int tid = threadIdx.x;
    lds[tid] = v;
    __syncthreads();
    for (int o = 1; o < kThreads; o <<= 1) {
        const T y = tid >= o ? lds[tid - o] : T(0);
        __syncthreads();
        lds[tid] += y;
        __syncthreads();
    }
    total = lds[kThreads - 1];
    v = tid ? lds[tid - 1] : T(0);
    __syncthreads();
    return v;
}

// A workgroup a row. What is kept is a run of the descending order: its last key, and how many entries of that key, by index.
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs p) {
    __shared__ double s_d[kThreads];
    __shared__ uint32_t s_u[kThreads];
    __shared__ uint32_t s_count[256];
    __shared__ unsigned long long s_mass[256];
    __shared__ uint32_t s_pick[3];
    __shared__ unsigned long long s_above;
    const int tid = threadIdx.x, r = blockIdx.x;
    const Row x = {static_cast<const char *>(p.logits) + r * p.stride * (p.io == TRHIP_F32 ? 4 : 2), p.io, p.vocab};
    uint32_t top = 0;
    for (int i = tid; i < p.vocab; i += kThreads) {
        const uint32_t k = x.key(i);
        top = k > top ? k : top;
    }
    s_u[tid] = top;
    __syncthreads();
    for (int o = kThreads / 2; o; o >>= 1) {
        if (tid < o) s_u[tid] = s_u[tid] > s_u[tid + o] ? s_u[tid] : s_u[tid + o];
        __syncthreads();
    }
    top = s_u[0];
    __syncthreads();
    if (top == 0) {
        if (tid == 0) {
            p.token[r] = -1;
            if (p.logprob) p.logprob[r] = __builtin_nanf("");
        }
        return;
    }
    const float t = p.temperature ? p.temperature[r] : 1.0f, tp = p.top_p ? p.top_p[r] : 1.0f, mp = p.min_p ? p.min_p[r] : 0.0f;
    const float u0 = p.u[r], u = u0 >= 0.0f ? u0 : 0.0f;
    const bool greedy = !(t > 0.0f);
    const int tk = greedy ? 1 : p.top_k ? p.top_k[r] : 0;
    const Weight w = {top, (double)of_key(top), greedy ? 1.0 : 1.0 / (double)t};
    uint32_t cut = 1, ties = 0xFFFFFFFFu;  // kept: keys above cut, and the first `ties` of cut
    int bits = 62;
    while ((p.vocab - 1) >> (62 - bits)) bits--;
    const double unit = ldexp(1.0, bits);
    for (int phase = 0; phase < 2; phase++) {
        double goal;  // entries, or weight, to reach
        if (phase == 0) {
            if (tk <= 0 || tk >= p.vocab) continue;
            goal = tk;
        } else {
            if (!(tp < 1.0f) || greedy) continue;
            double sum = 0;
            for (int i = tid; i < p.vocab; i += kThreads) {
                const uint32_t k = x.key(i);
                if (k > cut || (k == cut && ties == 0xFFFFFFFFu)) sum += w(k);
            }
            sum = sum_all(sum, s_d);
            if (ties != 0xFFFFFFFFu) sum += (double)ties * w(cut);
            goal = (double)tp * sum * unit;
        }
        uint32_t prefix = 0, mask = 0;
        unsigned long long above = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s_count[tid] = 0, s_mass[tid] = 0;
            __syncthreads();
            for (int i = tid; i < p.vocab; i += kThreads) {
                const uint32_t k = x.key(i);
                if ((k & mask) != prefix || k < cut) continue;
                const uint32_t b = k >> shift & 255;
                if (phase == 0) atomicAdd(&s_count[b], 1u);
                else if (k > cut || ties == 0xFFFFFFFFu) atomicAdd(&s_mass[b], (unsigned long long)rint(w(k) * unit));
            }
            __syncthreads();
            if (tid == 0) {
                if (phase == 1 && ties != 0xFFFFFFFFu && (cut & mask) == prefix) s_mass[cut >> shift & 255] += (unsigned long long)(rint(w(cut) * unit) * ties);
                unsigned long long run = above;
                int b = 255, pick = -1;
                unsigned long long pick_above = above;
                for (; b >= 0; b--) {
                    const unsigned long long n = phase == 0 ? s_count[b] : s_mass[b];
                    const bool some = phase == 0 ? n > 0 : n > 0;
                    if (some) pick = b, pick_above = run;
                    run += n;
                    if (some && (double)run >= goal) break;
                }
                s_pick[0] = pick < 0 ? 0 : pick;
                s_above = pick_above;
            }
            __syncthreads();
            above = s_above;
            prefix |= s_pick[0] << shift;
            mask |= 255u << shift;
            __syncthreads();
        }
        // of key `prefix` as many as it takes
        if (phase == 0) {
            cut = prefix;
            ties = (uint32_t)(tk - (int)above);
        } else {
            const double each = rint(w(prefix) * unit);
            double n = ceil((goal - (double)above) / each);
            n = n < 1 ? 1 : n;
            const uint32_t most = prefix == cut ? ties : 0xFFFFFFFFu;
            ties = n < (double)most ? (uint32_t)n : most;
            cut = prefix;
        }
    }
    const double low = mp >= 1.0f ? 1.0 : mp > 0.0f ? (double)mp : 0.0;
    if (greedy) ties = 1;
    // each thread's run of entries: how many of the cut's key, the kept weight, then the thread in which u falls
    const int each = (p.vocab + kThreads - 1) / kThreads, i0 = tid * each, i1 = i0 + each < p.vocab ? i0 + each : p.vocab;
    uint32_t eq = 0, total_eq;
    for (int i = i0; i < i1; i++) eq += x.key(i) == cut;
    const uint32_t eq0 = before_me(eq, s_u, total_eq);
    auto walk = [&](auto use) {
        uint32_t n = eq0;
        for (int i = i0; i < i1; i++) {
            const uint32_t k = x.key(i);
            const bool keep = k > cut || (k == cut && n < ties);
            n += k == cut;
            if (!keep || k == 0) continue;
            const double y = w(k);
            if (y >= low) use(i, y);
        }
    };
    double sum = 0, total;
    walk([&](int, double y) { sum += y; });
    const double start = before_me(sum, s_d, total);
    const double goal = (double)u * total;
    if (tid == 0) s_pick[0] = 0x7FFFFFFF, s_pick[1] = 0;
    __syncthreads();
    int found = 0x7FFFFFFF, last = -1;
    double run = start;
    walk([&](int i, double y) {
        run += y;
        if (y > 0) last = i;
        if (run > goal && found == 0x7FFFFFFF) found = i;
    });
    if (found != 0x7FFFFFFF) atomicMin(&s_pick[0], (uint32_t)found);
    if (last >= 0) atomicMax(&s_pick[1], (uint32_t)last);
    __syncthreads();
    if (tid == 0) {
        const int token = s_pick[0] != 0x7FFFFFFF ? (int)s_pick[0] : (int)s_pick[1];
        p.token[r] = token;
        if (p.logprob) p.logprob[r] = (float)log(w(x.key(token)) / total);
    }
}

}  // namespace

int launch_sample(trhip_ctx *ctx, const void *logits, int io, int64_t stride, int64_t rows, int64_t vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *u, int *token, float *logprob) {
    const SampleArgs p = {logits, io, stride, (int)vocab, temperature, top_k, top_p, min_p, u, token, logprob};
    hipLaunchKernelGGL(sample_kernel, dim3((unsigned)rows), dim3(kThreads), 0, ctx->stream, p);
    return launch_check(ctx, "sample");
}

}  // namespace trhip
