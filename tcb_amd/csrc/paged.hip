// paged.hip -- the bookkeeping of a paged key/value cache: the page tables of a batch, built from its requests' lengths,
// and the append of new key and value rows.
#include "trhip_internal.hpp"

namespace trhip {
namespace {

// Page tables. Request i holds old_i keys and brings add_i: have_i = ceil(old_i / page) pages it has, need_i =
// ceil((old_i + add_i) / page); the grow_i = need_i - have_i fresh ones are free[base_i ...], base the running sum of
// grow. One launch: every workgroup makes the running sums for itself (8 bytes a request, cached) and then writes its
// 4 x THREADS slots, four in a row a thread, whose request it finds by halving; the tables' fresh entries, lengths and starts are
// dealt over the workgroups by request. A slot's page is read from the table only where it was there before, else from
// the free list, so no workgroup waits for another's entries. What bounds it is latency: lengths, sums, one dependent read: 4.6 us
// in the kernel for 16 requests, 6.4 for 1024 of which 700 bring up to 511 tokens (10.1 with one slot a thread and sums through LDS).
// Sums saturate at 2^32 - 1 (a step of so many tokens has no slots anyway), so their order holds whatever the lengths are.
__device__ __forceinline__ int clamp31(uint32_t v) { return v > 0x7FFFFFFFu ? 0x7FFFFFFF : (int)v; }
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t running_sum(uint32_t v) {  // over the wave's lanes, inclusive
    v = sat_add(v, moved<0x111, 0xF>(v));  // row_shr 1, 2, 4, 8, then row_bcast 15 and 31
    v = sat_add(v, moved<0x112, 0xF>(v));
    v = sat_add(v, moved<0x114, 0xF>(v));
    v = sat_add(v, moved<0x118, 0xF>(v));
    v = sat_add(v, moved<0x142, 0xA>(v));
    return sat_add(v, moved<0x143, 0xC>(v));
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void page_tables_kernel(int nreq, int page_log2, const int *__restrict__ old_len,
                                                              const int *__restrict__ add_len, const int *__restrict__ free_list,
                                                              int64_t nfree, int *table, int64_t max_pages,
                                                              int *__restrict__ q_start, int *__restrict__ kv_len,
                                                              int *__restrict__ slots, int64_t nslots, int *__restrict__ used) {
    constexpr int WAVES = THREADS / 64, PER = 4;
    __shared__ uint32_t s_start[THREADS], s_base[THREADS], s_grow[THREADS];
    __shared__ int s_old[THREADS];  // -1: refused
    __shared__ uint32_t s_wave[2][WAVES];
    __shared__ int s_used[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t page = (int64_t)1 << page_log2, first = (int64_t)blockIdx.x * (PER * THREADS), mine = first + PER * tid;
    uint32_t tok0 = 0, base0 = 0;  // sums over the chunks of requests before this one
    int most = 0;
    int out[PER];
#pragma unroll
    for (int u = 0; u < PER; u++) out[u] = -1;
    for (int c = 0; c < nreq; c += THREADS) {
        const int i = c + tid;
        int old = 0, add = 0;
        if (i < nreq) {
            old = old_len[i];
            add = add_len[i];
            old = old < 0 ? 0 : old;
            add = add < 0 ? 0 : add;
        }
        const int64_t have = ((int64_t)old + page - 1) >> page_log2, need = ((int64_t)old + add + page - 1) >> page_log2;
        const uint32_t grow = need <= max_pages ? (uint32_t)(need - have) : 0;
        const uint32_t st = running_sum((uint32_t)add), sg = running_sum(grow);
        __syncthreads();  // the chunk before has been used
        if (lane == 63) {
            s_wave[0][w] = st;
            s_wave[1][w] = sg;
        }
        __syncthreads();
        uint32_t bt = tok0, bg = base0, tt = tok0, tg = base0;  // before this wave, after all
#pragma unroll
        for (int k = 0; k < WAVES; k++) {
            tt = sat_add(tt, s_wave[0][k]);
            tg = sat_add(tg, s_wave[1][k]);
            if (k < w) bt = tt, bg = tg;
        }
        const uint32_t end = sat_add(bt, st), start = end - (uint32_t)add, top = sat_add(bg, sg), base = top - grow;
        const bool fits = need <= max_pages && (grow == 0 || (int64_t)top <= nfree);
        if (fits && grow != 0 && (int64_t)top > most) most = (int)top;  // (one that needs no page fits behind any sum)
        s_start[tid] = start;
        s_old[tid] = fits ? old : -1;
        s_base[tid] = base;
        s_grow[tid] = fits ? grow : 0;
        // this workgroup's share of the requests' own outputs
        if (i < nreq && (int)((unsigned)(c / THREADS) % gridDim.x) == (int)blockIdx.x) {
            kv_len[i] = clamp31((uint32_t)old + (fits ? (uint32_t)add : 0u));
            q_start[i + 1] = clamp31(end);
            if (i == 0) q_start[0] = 0;
        }
        __syncthreads();
        const int cnt = nreq - c < THREADS ? nreq - c : THREADS;
        for (int k = (int)blockIdx.x * WAVES + w; k < cnt; k += (int)gridDim.x * WAVES) {  // a wave writes a request's fresh entries
            const uint32_t n = s_grow[k];
            if (n == 0) continue;
            int *row = table + (c + k) * max_pages + (((int64_t)s_old[k] + page - 1) >> page_log2);
            for (uint32_t j = lane; j < n; j += 64) row[j] = free_list[s_base[k] + j];
        }
        if (first < (int64_t)tt && first + PER * THREADS > (int64_t)tok0) {
            int lo = 0, hi = cnt;  // the last request that starts at or before this thread's first slot
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)s_start[mid] <= mine) lo = mid;
                else hi = mid;
            }
#pragma unroll
            for (int u = 0; u < PER; u++) {
                const int64_t t = mine + u;
                if (t < (int64_t)tok0 || t >= (int64_t)tt || t >= nslots) continue;
                while (lo + 1 < cnt && (int64_t)s_start[lo + 1] <= t) lo++;
                const int o = s_old[lo];
                if (o < 0) continue;
                const int64_t pos = (int64_t)o + (t - (int64_t)s_start[lo]), pi = pos >> page_log2, h = ((int64_t)o + page - 1) >> page_log2;
                int64_t pg = 0;
                if (pi < h) pg = table[(c + lo) * max_pages + pi];
                else pg = free_list[s_base[lo] + (pi - h)];
                const int64_t slot = (pg << page_log2) + (pos & (page - 1));
                if (slot >= 0 && slot <= 0x7FFFFFFF) out[u] = (int)slot;  // a page number out of range gives no slot
            }
        }
        tok0 = tt;
        base0 = tg;
    }
    if (mine + PER <= nslots && reinterpret_cast<uintptr_t>(slots) % 16 == 0) {
        *reinterpret_cast<int4 *>(slots + mine) = make_int4(out[0], out[1], out[2], out[3]);
    } else {
#pragma unroll
        for (int u = 0; u < PER; u++)
            if (mine + u < nslots) slots[mine + u] = out[u];
    }
    if (blockIdx.x == 0) {
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const int v = __shfl_xor(most, o);
            most = v > most ? v : most;
        }
        if (lane == 0) s_used[w] = most;
        __syncthreads();
        if (tid == 0) {
            for (int k = 1; k < WAVES; k++) most = s_used[k] > most ? s_used[k] : most;
            *used = most;
            if (nreq == 0) q_start[0] = 0;
        }
    }
}

// Cache append: eight elements a thread, rounded to the cache's type (nearest even) where the source's is another. It moves
// every element once, so its bytes bound it: 8192 tokens of 8 heads of 128 (67 MB read and written) take 12.9 us, 5.2 TB/s, part
// of it in the last cache; 16 tokens are a launch.
__device__ __forceinline__ uint4 take8(const void *src, int64_t at, int io, int dtype, bool wide) {
    uint32_t h[8];
    if (io == TRHIP_F32) {
        const float *s = static_cast<const float *>(src) + at;
        float f[8];
        if (wide) {
            *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(s);
            *reinterpret_cast<float4 *>(f + 4) = *reinterpret_cast<const float4 *>(s + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = s[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = f32_to_h16(f[i], dtype);
    } else {
        const uint16_t *s = static_cast<const uint16_t *>(src) + at;
        if (io == dtype && wide) return *reinterpret_cast<const uint4 *>(s);
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = io == dtype ? (uint32_t)s[i] : f32_to_h16(h16_to_f32(s[i], io), dtype);
    }
    return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}
__global__ __launch_bounds__(256) void kv_append_kernel(uint16_t *__restrict__ kc, uint16_t *__restrict__ vc, int dtype, int page_log2,
                                                        int64_t places, int heads, int dim, int64_t tokens, const void *__restrict__ k,
                                                        const void *__restrict__ v, int io, int64_t stride,
                                                        const int *__restrict__ slots, int wide) {
    const int row = heads * dim / 8, per = 2 * row;  // eights of a token: k's, then v's
    const int64_t total = tokens * per, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t x = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; x < total; x += step) {
        const int64_t t = x / per;
        const int c = (int)(x - t * per), e = c < row ? c : c - row;
        const int64_t slot = slots[t];
        if ((uint64_t)slot >= (uint64_t)places) continue;
        const int head = 8 * e / dim, d = 8 * e - head * dim;
        const int64_t pg = slot >> page_log2, in = slot & ((1 << page_log2) - 1);
        const uint4 y = take8(c < row ? k : v, t * stride + 8 * e, io, dtype, wide);
        *reinterpret_cast<uint4 *>((c < row ? kc : vc) + (((pg * heads + head) << page_log2) + in) * dim + d) = y;
    }
}

}  // namespace

int launch_page_tables(trhip_ctx *ctx, int64_t nreq, int page, const int *old_len, const int *add_len, const int *free_list,
                       int64_t nfree, int *table, int64_t max_pages, int *q_start, int *kv_len, int *slots, int64_t nslots,
                       int *used) {
    const int lg = __builtin_ctz((unsigned)page);
    // (16 requests in workgroups of 256 threads, 1024 in ones of 1024: one chunk of lengths either way)
    const int64_t threads = nreq <= 256 ? 256 : 1024, grid = nslots > 0 ? (nslots + 4 * threads - 1) / (4 * threads) : 1;
    if (grid >= ((int64_t)1 << 31)) return fail(ctx, TRHIP_ERR_INVALID, "page_tables: too many slots");
    if (threads == 256)
        hipLaunchKernelGGL(page_tables_kernel<256>, dim3((unsigned)grid), dim3(256), 0, ctx->stream, (int)nreq, lg, old_len, add_len,
                           free_list, nfree, table, max_pages, q_start, kv_len, slots, nslots, used);
    else
        hipLaunchKernelGGL(page_tables_kernel<1024>, dim3((unsigned)grid), dim3(1024), 0, ctx->stream, (int)nreq, lg, old_len, add_len,
                           free_list, nfree, table, max_pages, q_start, kv_len, slots, nslots, used);
    return launch_check(ctx, "page_tables");
}

int launch_kv_append(trhip_ctx *ctx, const trhip_kv *kv, int64_t tokens, const void *k, const void *v, int io, int64_t stride,
                     const int *slots) {
    const int64_t esize = io == TRHIP_F32 ? 4 : 2;
    const int wide = reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && stride * esize % 16 == 0;
    const int64_t total = tokens * (kv->heads * kv->dim / 4);
    int64_t blocks = (total + 255) / 256;
    const int64_t cap = (int64_t)(ctx->sm_count > 0 ? ctx->sm_count : 256) * 16;
    if (blocks > cap) blocks = cap;
    hipLaunchKernelGGL(kv_append_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, static_cast<uint16_t *>(kv->k),
                       static_cast<uint16_t *>(kv->v), kv->dtype, __builtin_ctz((unsigned)kv->page), kv->pages * kv->page, kv->heads,
                       kv->dim, tokens, k, v, io, stride, slots, wide);
    return launch_check(ctx, "kv_append");
}

}  // namespace trhip
