// Pooled embedding lookup with scaling, and its gradient by sorted tokens.
//
//   p_b = s c_b sum_{t in bag b} w_t E[id_t]        c_b = 1 | 1/n_b | 1/sqrt(n_b)
//   y_b = p_b / |p_b|  (or p_b)
//   dp_b = k_b (g_b - y_b <g_b, y_b>)               k_b = s c_b / |p_b|   (k_b g_b with k_b = s c_b when not normalised)
//   dE[v] = sum_{t: id_t = v} w_t dp_{b(t)}         dw_t = <dp_{b(t)}, E[id_t]>
//
// Both sums are one operation, a segmented sum of gathered, weighted rows: forward the segments are the bags and the rows
// come from the table; backward the segments are the runs of equal tokens among the occurrences sorted by (token,
// position) and the rows are the bags' dp.  k_segsum walks equal shares of the positions whatever the segments' lengths;
// a segment that crosses a share's border leaves partial sums that k_segjoin adds in the order of the positions.  No
// atomics: the same inputs give the same bits.
//
// Stands in front of retriever/hybrid_search.py:60-64 of the reference, which embeds the query text before the search.
#include <algorithm>
#include <initializer_list>

#include "crag_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

__device__ __forceinline__ float bf16_f32(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
__device__ __forceinline__ uint32_t f32_bf16(float f) {  // round to nearest even; a NaN stays one
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// VEC consecutive elements of a row (aligned to VEC elements or 16 bytes)
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* p, long long i, float (&x)[VEC]) {
    if constexpr (DT == CRAG_F32) {
        const float* f = (const float*)p + i;
        if constexpr (VEC % 4 == 0) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const f32x4_t v = *(const f32x4_t*)(f + j);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[j + k] = v[k];
            }
        } else if constexpr (VEC == 2) {
            const f32x2_t v = *(const f32x2_t*)f;
            x[0] = v[0];
            x[1] = v[1];
        } else {
            x[0] = *f;
        }
    } else {
        const unsigned short* h = (const unsigned short*)p + i;
        if constexpr (VEC == 8) {
            const u32x4_t v = *(const u32x4_t*)h;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[2 * k] = bf16_f32(v[k] & 0xffffu);
                x[2 * k + 1] = bf16_f32(v[k] >> 16);
            }
        } else if constexpr (VEC == 2) {
            const uint32_t v = *(const uint32_t*)h;
            x[0] = bf16_f32(v & 0xffffu);
            x[1] = bf16_f32(v >> 16);
        } else if constexpr (VEC == 4) {
            const uint2 v = *(const uint2*)h;
            x[0] = bf16_f32(v.x & 0xffffu);
            x[1] = bf16_f32(v.x >> 16);
            x[2] = bf16_f32(v.y & 0xffffu);
            x[3] = bf16_f32(v.y >> 16);
        } else {
            x[0] = bf16_f32(*h);
        }
    }
}
template <int VEC>
__device__ __forceinline__ void store_vec(void* p, int dt, long long i, const float (&x)[VEC]) {
    if (dt == CRAG_F32) {
        float* f = (float*)p + i;
        if constexpr (VEC % 4 == 0) {
#pragma unroll
            for (int k = 0; k < VEC; k += 4) *(f32x4_t*)(f + k) = (f32x4_t){x[k], x[k + 1], x[k + 2], x[k + 3]};
        } else if constexpr (VEC == 2) {
            *(f32x2_t*)f = (f32x2_t){x[0], x[1]};
        } else {
            *f = x[0];
        }
    } else {
        unsigned short* h = (unsigned short*)p + i;
        if constexpr (VEC >= 2) {
#pragma unroll
            for (int k = 0; k < VEC; k += 2) *(uint32_t*)(h + k) = f32_bf16(x[k]) | (f32_bf16(x[k + 1]) << 16);
        } else {
            *h = (unsigned short)f32_bf16(x[0]);
        }
    }
}

// A row is held by `lpr` lanes (8 .. 64, a power of two), NV pieces of VEC elements in each: lane `sub` holds elements
// (n * lpr + sub) * VEC ..., n < NV.
template <int VEC, int NV>
struct Row {
    float x[NV][VEC];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[n][k] = 0.f;
    }
    template <int DT>
    __device__ __forceinline__ void load(const void* base, long long row, int dim, int lpr, int sub, bool on) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int e = (n * lpr + sub) * VEC;
            if (on && e < dim) {
                load_vec<DT, VEC>(base, row * dim + e, x[n]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) x[n][k] = 0.f;
            }
        }
    }
    __device__ __forceinline__ void fma(const Row& o, float w) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[n][k] = fmaf(o.x[n][k], w, x[n][k]);
    }
    __device__ __forceinline__ void add(const Row& o) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[n][k] += o.x[n][k];
    }
    __device__ __forceinline__ void store(void* base, int dt, long long row, int dim, int lpr, int sub) const {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int e = (n * lpr + sub) * VEC;
            if (e < dim) store_vec<VEC>(base, dt, row * dim + e, x[n]);
        }
    }
};

// Last entry of off[0 .. n] that is <= p, as its index (-1: none)
__device__ __forceinline__ int last_le(const long long* __restrict__ off, int n, long long p) {
    int lo = -1, hi = n + 1;
    while (hi - lo > 1) {
        const int mid = (int)(((long long)lo + hi) >> 1);
        if (off[mid] <= p) lo = mid; else hi = mid;
    }
    return lo;
}

// A finished segment's epilogue: forward scale, pool factor, norm and coefficient; backward nothing.  All lanes of the row.
template <bool BWD, int VEC, int NV>
__device__ __forceinline__ void finish(const CragSegArgs& a, long long seg, Row<VEC, NV>& r, int count, int sub) {
    if constexpr (!BWD) {
        float f = a.scale;
        if (a.mode == CRAG_POOL_MEAN) f = (float)((double)a.scale / (count > 0 ? count : 1));
        if (a.mode == CRAG_POOL_SQRT) f = (float)((double)a.scale / sqrt((double)(count > 0 ? count : 1)));
        float coef = f;
        if (a.normalize) {
            // |p| in float64: squares of float32 neither overflow nor vanish there
            double ss = 0.0;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int k = 0; k < VEC; ++k) ss += (double)r.x[n][k] * (double)r.x[n][k];
            for (int o = a.lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
            const double s = sqrt(ss);  // of the unscaled sum: y = sign(f) * sum / |sum|
            const double inv = s > 0.0 && f != 0.f ? (f < 0.f ? -1.0 : 1.0) / s : 0.0 * s;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int k = 0; k < VEC; ++k) r.x[n][k] = (float)((double)r.x[n][k] * inv);
            coef = (float)inv;  // s c_b / |s c_b sum|
        } else {
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int k = 0; k < VEC; ++k) r.x[n][k] *= f;
        }
        if (a.coef && sub == 0) a.coef[seg] = coef;
    }
    r.store(a.out, a.out_dtype, seg, a.dim, a.lpr, sub);
}

// One group of lpr lanes walks the positions [g * share, (g + 1) * share).
template <int DT, bool BWD, int VEC, int NV>
__global__ __launch_bounds__(256) void k_segsum(CragSegArgs a) {
    constexpr int U = NV * VEC <= 8 ? 8 : 4;  // rows in flight
    const int lane = threadIdx.x & 63;
    const int lpr = a.lpr, sub = lane & (lpr - 1), first = lane & ~(lpr - 1);
    const long long g = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / lpr) + lane / lpr;
    const long long T = a.n;
    long long p0 = g * a.share;
    long long p1 = p0 + a.share < T ? p0 + a.share : T;
    if (p0 > T) p0 = p1 = T;
    // forward: the bags cover [lo, hi)
    long long lo = 0, hi = T, end = 0;
    long long seg = -1;       // segment the running sum belongs to
    bool before = false;      // ... and it has positions in front of this share
    int count = 0;
    long long head = -1, tail = -1;
    if constexpr (!BWD) {
        lo = a.offsets[0];
        hi = a.offsets[a.n_seg];
        lo = lo < 0 ? 0 : lo;
        hi = hi > T ? T : hi;
    }
    Row<VEC, NV> acc;
    acc.zero();
    auto partial = [&](int which) {
        acc.store(a.partial, CRAG_F32, 2 * g + which, a.dim, lpr, sub);
        if (sub == 0) a.partial_count[2 * g + which] = count;
        (which == 0 ? head : tail) = seg;
    };
    for (long long base = p0; base < p0 + a.share; base += lpr) {  // the same number of rounds in every group
        // what each position of the round reads: lane `sub` looks up position base + sub
        const long long pm = base + sub;
        int row = -1, key = -1;
        float w = 0.f;
        if (pm < p1) {
            if constexpr (BWD) {
                key = (int)a.keys[pm];
                if (key < a.vocab) {
                    const uint32_t t = a.perm[pm];
                    row = a.bag[t];
                    w = a.weights ? a.weights[t] : 1.f;
                } else {
                    key = -1;
                }
            } else if (pm >= lo && pm < hi) {
                const int id = a.ids[pm];
                if (id >= 0 && id < a.vocab) {
                    row = id;
                    w = a.weights ? a.weights[pm] : 1.f;
                }
            }
        }
        const int rounds = a.share < lpr ? a.share : lpr;
        for (int j = 0; j < rounds; j += U) {
            Row<VEC, NV> x[U];
            float wu[U];
            int ru[U], ku[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ru[u] = __shfl(row, first + j + u);
                wu[u] = __shfl(w, first + j + u);
                if constexpr (BWD) ku[u] = __shfl(key, first + j + u);
                x[u].template load<DT>(a.src, ru[u], a.dim, lpr, sub, ru[u] >= 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long p = base + j + u;
                if (p >= p1) continue;
                if constexpr (BWD) {
                    const int k = ku[u];
                    if (k != (int)seg || p == p0) {
                        if (p != p0 && seg >= 0) {
                            if (before) partial(0); else finish<BWD>(a, seg, acc, count, sub);
                        }
                        before = p == p0 && p > 0 && k >= 0 && (int)a.keys[p - 1] == k;
                        seg = k;
                        acc.zero();
                    }
                    if (k >= 0) acc.fma(x[u], wu[u]);
                } else {
                    if (p < lo || p >= hi) continue;
                    if (seg < 0 || p >= end) {
                        if (seg >= 0) {
                            if (before) partial(0); else finish<BWD>(a, seg, acc, count, sub);
                        }
                        seg = last_le(a.offsets, a.n_seg, p);
                        if (seg >= a.n_seg) { seg = -1; hi = p; continue; }
                        end = a.offsets[seg + 1];
                        before = a.offsets[seg] < p0 && p == p0;
                        count = 0;
                        acc.zero();
                    }
                    if (ru[u] >= 0) {
                        acc.fma(x[u], wu[u]);
                        ++count;
                    }
                }
            }
        }
    }
    if (seg >= 0) {
        bool after;
        if constexpr (BWD) after = p1 < T && (int)a.keys[p1] == (int)seg;
        else after = p1 < hi && end > p1;
        if (before) partial(0);
        else if (after) partial(1);
        else finish<BWD>(a, seg, acc, count, sub);
    }
    if (sub == 0 && g < a.n_share) {
        a.partial_seg[2 * g] = (int)head;
        a.partial_seg[2 * g + 1] = (int)tail;
    }
}

// Blocks [0, n_share): the segment whose first partial sum is share g's tail -- it goes on through the heads of the shares
// behind it.  Blocks behind that: forward, the bags without positions.
template <bool BWD, int VEC, int NV>
__global__ __launch_bounds__(256) void k_segjoin(CragSegArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    float* part = (float*)smem;  // [256 / lpr][dim of a row as held: lpr * VEC * NV]
    __shared__ int s_end, s_count;
    const int tid = threadIdx.x, lpr = a.lpr, sub = tid & (lpr - 1), grp = tid / lpr, groups = 256 / lpr;
    if ((long long)blockIdx.x >= a.n_share) {
        if constexpr (!BWD) {
            const long long stride = (long long)(gridDim.x - a.n_share) * groups;
            for (long long b = ((long long)blockIdx.x - a.n_share) * groups + grp; b < a.n_seg; b += stride) {
                long long x0 = a.offsets[b], x1 = a.offsets[b + 1];
                x0 = x0 < 0 ? 0 : x0;
                x1 = x1 > a.n ? a.n : x1;
                if (x0 < x1) continue;
                Row<VEC, NV> r;
                r.zero();
                finish<BWD>(a, b, r, 0, sub);
            }
        }
        return;
    }
    const long long g = blockIdx.x;
    const int seg = a.partial_seg[2 * g + 1];
    if (seg < 0) return;
    if (tid == 0) {
        s_end = 0x7fffffff;
        s_count = 0;
    }
    __syncthreads();
    // the last share that holds a head of this segment
    for (long long j0 = g + 1;; j0 += 256) {
        const long long j = j0 + tid;
        if (j >= a.n_share || a.partial_seg[2 * j] != seg) atomicMin(&s_end, (int)(j < a.n_share ? j : a.n_share));
        __syncthreads();
        if (s_end != 0x7fffffff) break;
        __syncthreads();
    }
    const int n = s_end - (int)g;  // partial sums: tail of g, heads of g + 1 .. s_end - 1
    Row<VEC, NV> acc;
    acc.zero();
    int count = 0;
    const int per = (n + groups - 1) / groups;
    const int i0 = grp * per, i1 = i0 + per < n ? i0 + per : n;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
        const long long slot = i == 0 ? 2 * g + 1 : 2 * (g + i);
        Row<VEC, NV> x;
        x.template load<CRAG_F32>(a.partial, slot, a.dim, lpr, sub, true);
        acc.add(x);
        count += a.partial_count[slot];
    }
    if (!BWD && sub == 0 && count) atomicAdd(&s_count, count);
    const int rowlen = lpr * VEC * NV;
    if (grp > 0) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int k = 0; k < VEC; ++k) part[grp * rowlen + (v * lpr + sub) * VEC + k] = acc.x[v][k];
    }
    __syncthreads();
    if (grp == 0) {
        for (int o = 1; o < groups && o * per < n; ++o)
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc.x[v][k] += part[o * rowlen + (v * lpr + sub) * VEC + k];
        finish<BWD>(a, seg, acc, s_count, sub);
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// dp_b = coef_b (g_b - y_b <g_b, y_b>), or coef_b g_b.  One wave per bag.
__global__ __launch_bounds__(256) void k_embed_dpool(const float* __restrict__ grad, const float* __restrict__ y,
                                                     const float* __restrict__ coef, int n_bags, int dim, int normalize,
                                                     float* __restrict__ dp) {
    const int lane = threadIdx.x & 63;
    const long long b = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= n_bags) return;
    const float* g = grad + b * dim;
    const float* yb = y + b * dim;
    double dot = 0.0;
    if (normalize) {
        for (int d = lane; d < dim; d += 64) dot += (double)g[d] * (double)yb[d];
        for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o);
    }
    const float c = coef[b];
    for (int d = lane; d < dim; d += 64) {
        const double v = normalize ? (double)g[d] - (double)yb[d] * dot : (double)g[d];
        dp[b * dim + d] = (float)(v * (double)c);
    }
}

// bag[t] of every position (-1 outside every bag); the sort's first keys and payload
__global__ __launch_bounds__(256) void k_embed_bag_of(const int* __restrict__ ids, long long n, const long long* __restrict__ offsets,
                                                      int n_bags, int vocab, int* __restrict__ bag, uint32_t* __restrict__ keys,
                                                      uint32_t* __restrict__ perm) {
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t >= n) return;
    int b = last_le(offsets, n_bags, t);
    if (b >= n_bags) b = -1;
    bag[t] = b;
    const int id = ids[t];
    keys[t] = b >= 0 && id >= 0 && id < vocab ? (uint32_t)id : (uint32_t)vocab;
    perm[t] = (uint32_t)t;
}

// up to SORT_SMALL positions: one workgroup sorts (key, position) in LDS
constexpr int SORT_SMALL = 8192;
__global__ __launch_bounds__(1024) void k_sort_small(uint32_t* __restrict__ keys, uint32_t* __restrict__ perm, int n, int P) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    unsigned long long* s = (unsigned long long*)smem;
    for (int i = threadIdx.x; i < P; i += 1024) s[i] = i < n ? ((unsigned long long)keys[i] << 32) | (uint32_t)i : ~0ull;
    __syncthreads();
    for (int k = 2; k <= P; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < (P >> 1); i += 1024) {
                const int x = ((i & ~(j - 1)) << 1) | (i & (j - 1)), y = x | j;
                const bool up = (x & k) == 0;
                const unsigned long long u = s[x], v = s[y];
                if ((u > v) == up) {
                    s[x] = v;
                    s[y] = u;
                }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < n; i += 1024) {
        keys[i] = (uint32_t)(s[i] >> 32);
        perm[i] = (uint32_t)s[i];
    }
}

// Stable least-significant-digit radix sort, 8 bits a pass: counts per tile, prefix per digit, ordered scatter.
constexpr int SORT_TILE = 4096, SORT_PER = SORT_TILE / 256;
__global__ __launch_bounds__(256) void k_sort_count(const uint32_t* __restrict__ keys, long long n, int shift, int tiles,
                                                    uint32_t* __restrict__ hist) {
    __shared__ uint32_t h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE;
#pragma unroll
    for (int i = 0; i < SORT_PER; ++i) {
        const long long p = base + i * 256 + threadIdx.x;
        if (p < n) atomicAdd(&h[(keys[p] >> shift) & 255u], 1u);
    }
    __syncthreads();
    hist[(long long)threadIdx.x * tiles + blockIdx.x] = h[threadIdx.x];
}
// block d: exclusive prefix of digit d's counts over the tiles, its total behind them
__global__ __launch_bounds__(256) void k_sort_prefix(uint32_t* __restrict__ hist, int tiles, uint32_t* __restrict__ total) {
    __shared__ uint32_t ws[4];
    uint32_t* h = hist + (long long)blockIdx.x * tiles;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    uint32_t run = 0;
    for (int t0 = 0; t0 < tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        const uint32_t c = t < tiles ? h[t] : 0u;
        uint32_t inc = c;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 63) ws[wv] = inc;
        __syncthreads();
        uint32_t base = run;
        for (int w = 0; w < wv; ++w) base += ws[w];
        if (t < tiles) h[t] = base + inc - c;
        run += ws[0] + ws[1] + ws[2] + ws[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) total[blockIdx.x] = run;
}
__global__ __launch_bounds__(256) void k_sort_scatter(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ perm, long long n,
                                                      int shift, int tiles, const uint32_t* __restrict__ hist,
                                                      const uint32_t* __restrict__ total, uint32_t* __restrict__ keys_out,
                                                      uint32_t* __restrict__ perm_out) {
    __shared__ uint32_t cnt[4][256];  // per wave: counts of its quarter of the tile, then where its next key of a digit goes
    __shared__ uint32_t ws[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    for (int w = 0; w < 4; ++w) cnt[w][tid] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * SORT_TILE + wv * (SORT_TILE / 4);
    uint32_t k[SORT_PER], v[SORT_PER];
#pragma unroll
    for (int i = 0; i < SORT_PER; ++i) {
        const long long p = base + i * 64 + lane;
        k[i] = p < n ? keys[p] : 0u;
        v[i] = p < n ? perm[p] : 0u;
        if (p < n) atomicAdd(&cnt[wv][(k[i] >> shift) & 255u], 1u);
    }
    // where digit tid starts: all smaller digits, then this digit in the tiles in front
    const uint32_t tot = total[tid];
    uint32_t inc = tot;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 63) ws[wv] = inc;
    __syncthreads();
    uint32_t at = inc - tot + hist[(long long)tid * tiles + blockIdx.x];
    for (int w = 0; w < wv; ++w) at += ws[w];
    for (int w = 0; w < 4; ++w) {
        const uint32_t c = cnt[w][tid];
        cnt[w][tid] = at;
        at += c;
    }
    __syncthreads();
    volatile uint32_t* next = cnt[wv];
#pragma unroll
    for (int i = 0; i < SORT_PER; ++i) {
        const long long p = base + i * 64 + lane;
        const bool on = p < n;
        const uint32_t d = (k[i] >> shift) & 255u;
        unsigned long long same = __ballot(on);
#pragma unroll
        for (int bit = 0; bit < 8; ++bit) {
            const unsigned long long m = __ballot((d >> bit) & 1u);
            same &= (d >> bit) & 1u ? m : ~m;
        }
        const uint32_t rank = __popcll(same & ((1ull << lane) - 1ull));
        uint32_t where = 0;
        if (on) where = next[d];
        __builtin_amdgcn_wave_barrier();
        if (on && rank == 0) next[d] = where + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (on) {
            keys_out[where + rank] = k[i];
            perm_out[where + rank] = v[i];
        }
    }
}

// dw_t = <dp_b, E[id_t]>; groups of lpr lanes over shares of the positions, as k_segsum
template <int DT, int VEC, int NV>
__global__ __launch_bounds__(256) void k_embed_dweights(CragSegArgs a, const void* __restrict__ table, const int* __restrict__ ids,
                                                        float* __restrict__ dw) {
    constexpr int U = NV * VEC <= 8 ? 8 : 4;
    const int lane = threadIdx.x & 63;
    const int lpr = a.lpr, sub = lane & (lpr - 1), first = lane & ~(lpr - 1);
    const long long g = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / lpr) + lane / lpr;
    const long long p0 = g * a.share, p1 = p0 + a.share < a.n ? p0 + a.share : a.n;
    int cur = -1;
    Row<VEC, NV> d;
    d.zero();
    for (long long base = p0; base < p0 + a.share; base += lpr) {
        const long long pm = base + sub;
        int id = -1, bag = -1;
        if (pm < p1) {
            bag = a.bag[pm];
            id = ids[pm];
            if (bag < 0 || id < 0 || id >= a.vocab) id = -1;
        }
        float mine = 0.f;
        const int rounds = a.share < lpr ? a.share : lpr;
        for (int j = 0; j < rounds; j += U) {
            Row<VEC, NV> x[U];
            int bu[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int id_u = __shfl(id, first + j + u);
                bu[u] = __shfl(bag, first + j + u);
                if (id_u < 0) bu[u] = -1;
                x[u].template load<DT>(table, id_u, a.dim, lpr, sub, id_u >= 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (bu[u] >= 0 && bu[u] != cur) {
                    cur = bu[u];
                    d.template load<CRAG_F32>(a.src, cur, a.dim, lpr, sub, true);
                }
                float s = 0.f;
                if (bu[u] >= 0) {
#pragma unroll
                    for (int n = 0; n < NV; ++n)
#pragma unroll
                        for (int k = 0; k < VEC; ++k) s = fmaf(x[u].x[n][k], d.x[n][k], s);
                }
                for (int o = lpr >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o);
                if (sub == j + u) mine = s;
            }
        }
        if (pm < p1) dw[pm] = mine;
    }
}

__global__ __launch_bounds__(256) void k_fill_rows(u32x4_t* __restrict__ out, long long n16, unsigned char* __restrict__ rest, int n_rest) {
    const long long stride = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n16; i += stride) out[i] = (u32x4_t){0, 0, 0, 0};
    if (blockIdx.x == 0 && (int)threadIdx.x < n_rest) rest[threadIdx.x] = 0;
}

__global__ __launch_bounds__(256) void k_zero_f32(float* __restrict__ out, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = 0.f;
}

// ---- geometry ------------------------------------------------------------------------------------------------------------
struct Shape {
    int vec, nv, lpr;
};
// lanes per row and pieces per lane: the fewest idle lanes, then the most lanes
Shape row_shape(int dim, int vec) {
    const int pieces = (dim + vec - 1) / vec;
    static const int kNv[] = {1, 2, 3, 4, 8, 16, 32};
    Shape best = {vec, 0, 0};
    int best_held = 0x7fffffff;
    for (int lpr = 64; lpr >= 8; lpr >>= 1)
        for (int nv : kNv) {
            if (nv * vec > 32) continue;
            if (lpr * nv < pieces) continue;
            if (lpr * nv < best_held) {
                best_held = lpr * nv;
                best.nv = nv;
                best.lpr = lpr;
            }
            break;
        }
    return best;
}
int vec_of(int dim, int esz, std::initializer_list<const void*> ptrs) {
    for (int vec : {esz == 2 ? 8 : 4, 2}) {
        bool ok = dim % vec == 0;
        for (const void* p : ptrs) ok = ok && ((uintptr_t)p % (size_t)(vec * esz > 16 ? 16 : vec * esz)) == 0;
        if (ok) return vec;
    }
    return 1;
}
// positions a group of lanes walks: shares enough to fill the chip several times over, but not so many that joining the
// segments that cross their borders weighs against the sums themselves
int share_of(long long n, int lpr) {
    const long long groups = 256ll * 16 * (64 / lpr);
    int c = 8;
    while (c < 256 && n / c > groups) c <<= 1;
    return c;
}

#define CRAG_SEG_CASES(X) \
    X(8, 1) X(8, 2) X(8, 3) X(8, 4) X(4, 1) X(4, 2) X(4, 3) X(4, 4) X(4, 8) X(2, 1) X(2, 2) X(2, 3) X(2, 4) X(2, 8) X(2, 16) \
    X(1, 1) X(1, 2) X(1, 3) X(1, 4) X(1, 8) X(1, 16) X(1, 32)

template <int DT, bool BWD>
int launch_segsum(const CragSegArgs& a, const Shape& sh, hipStream_t s) {
    const long long blocks = (a.n_share + 4 * (64 / sh.lpr) - 1) / (4 * (64 / sh.lpr));
    long long empties = 0;
    if (!BWD) empties = std::min<long long>(512, (a.n_seg + 255) / 256);
    const size_t lds = sizeof(float) * 256 * sh.vec * sh.nv;
#define X(V, N)                                                                                                                \
    if (sh.vec == V && sh.nv == N) {                                                                                           \
        if constexpr (!(DT == CRAG_F32 && V == 8)) {                                                                           \
            if (blocks) hipLaunchKernelGGL((k_segsum<DT, BWD, V, N>), dim3((unsigned)blocks), dim3(256), 0, s, a);              \
            if (a.n_share + empties)                                                                                           \
                hipLaunchKernelGGL((k_segjoin<BWD, V, N>), dim3((unsigned)(a.n_share + empties)), dim3(256), lds, s, a);         \
            return (int)hipGetLastError();                                                                                     \
        }                                                                                                                      \
    }
    CRAG_SEG_CASES(X)
#undef X
    return -1;
}
template <int DT>
int launch_dweights(const CragSegArgs& a, const Shape& sh, const void* table, const int* ids, float* dw, hipStream_t s) {
    const long long blocks = (a.n_share + 4 * (64 / sh.lpr) - 1) / (4 * (64 / sh.lpr));
    if (!blocks) return 0;
#define X(V, N)                                                                                                            \
    if (sh.vec == V && sh.nv == N) {                                                                                       \
        if constexpr (!(DT == CRAG_F32 && V == 8)) {                                                                       \
            hipLaunchKernelGGL((k_embed_dweights<DT, V, N>), dim3((unsigned)blocks), dim3(256), 0, s, a, table, ids, dw);   \
            return (int)hipGetLastError();                                                                                 \
        }                                                                                                                  \
    }
    CRAG_SEG_CASES(X)
#undef X
    return -1;
}

struct Carve {
    char* p;
    size_t used = 0;
    void* take(size_t bytes) {
        void* r = p ? p + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        return r;
    }
};
// most shares any alignment of the pointers can lead to (the workspace is sized without them)
long long most_shares(long long n, int dim) {
    long long most = 1;
    for (int vec : {1, 2, 4, 8}) {
        const Shape sh = row_shape(dim, vec);
        const int share = share_of(n, sh.lpr);
        most = std::max(most, (n + share - 1) / share);
    }
    return most;
}

struct SegWs {
    float* partial;
    int *partial_seg, *partial_count;
};
SegWs carve_seg(Carve& c, long long n, int dim) {
    const size_t slots = 2 * (size_t)most_shares(n, dim);
    SegWs w;
    w.partial = (float*)c.take(sizeof(float) * slots * (size_t)dim);
    w.partial_seg = (int*)c.take(sizeof(int) * slots);
    w.partial_count = (int*)c.take(sizeof(int) * slots);
    return w;
}
struct BwdWs {
    SegWs seg;
    float* dp;
    int* bag;
    uint32_t *keys[2], *perm[2], *hist, *total;
};
BwdWs carve_bwd(Carve& c, long long n, int n_bags, int dim) {
    BwdWs w;
    w.seg = carve_seg(c, n, dim);
    w.dp = (float*)c.take(sizeof(float) * (size_t)n_bags * (size_t)dim);
    w.bag = (int*)c.take(sizeof(int) * (size_t)n);
    for (int i = 0; i < 2; ++i) {
        w.keys[i] = (uint32_t*)c.take(sizeof(uint32_t) * (size_t)n);
        w.perm[i] = (uint32_t*)c.take(sizeof(uint32_t) * (size_t)n);
    }
    w.hist = (uint32_t*)c.take(sizeof(uint32_t) * 256 * (size_t)((n + SORT_TILE - 1) / SORT_TILE));
    w.total = (uint32_t*)c.take(sizeof(uint32_t) * 256);
    return w;
}

}  // namespace

size_t crag_embed_ws_bytes(long long n, int n_bags, int dim, bool backward) {
    Carve c{nullptr};
    if (backward) carve_bwd(c, n, n_bags, dim);
    else carve_seg(c, n, dim);
    return c.used;
}

int crag_launch_embed_forward(const CragEmbedArgs& e, hipStream_t s) {
    Carve c{(char*)e.workspace};
    const SegWs w = carve_seg(c, e.n, e.dim);
    const int esz = e.dtype == CRAG_F32 ? 4 : 2;
    int vec = vec_of(e.dim, esz, {e.table});
    const int osz = e.out_dtype == CRAG_F32 ? 4 : 2;
    while (vec > 1 && ((uintptr_t)e.out % (size_t)std::min(16, vec * osz))) vec = vec > 2 ? 2 : 1;
    const Shape sh = row_shape(e.dim, vec);
    CragSegArgs a = {};
    a.src = e.table;
    a.n = e.n;
    a.n_seg = e.n_bags;
    a.dim = e.dim;
    a.vocab = (int)e.vocab;
    a.lpr = sh.lpr;
    a.share = share_of(e.n, sh.lpr);
    a.n_share = (e.n + a.share - 1) / a.share;
    a.ids = e.ids;
    a.weights = e.weights;
    a.offsets = e.offsets;
    a.partial = w.partial;
    a.partial_seg = w.partial_seg;
    a.partial_count = w.partial_count;
    a.out = e.out;
    a.out_dtype = e.out_dtype;
    a.mode = e.mode;
    a.normalize = e.normalize;
    a.scale = e.scale;
    a.coef = e.coef;
    return e.dtype == CRAG_F32 ? launch_segsum<CRAG_F32, false>(a, sh, s) : launch_segsum<CRAG_BF16, false>(a, sh, s);
}

int crag_launch_embed_backward(const CragEmbedArgs& args, hipStream_t s) {
    CragEmbedArgs e = args;
    Carve c{(char*)e.workspace};
    const BwdWs w = carve_bwd(c, e.n, e.n_bags, e.dim);
    const int esz = e.dtype == CRAG_F32 ? 4 : 2;
    int rc;
    if (e.n_bags == 0) {  // every position is outside every bag
        if (e.d_weights && e.n > 0) hipLaunchKernelGGL(k_zero_f32, dim3((unsigned)((e.n + 255) / 256)), dim3(256), 0, s, e.d_weights, e.n);
        e.n = 0;
    }
    if (e.n_bags > 0)
        hipLaunchKernelGGL(k_embed_dpool, dim3((unsigned)((e.n_bags + 3) / 4)), dim3(256), 0, s, e.grad, e.y, e.coef, e.n_bags, e.dim,
                           e.normalize, w.dp);
    if (e.n > 0)
        hipLaunchKernelGGL(k_embed_bag_of, dim3((unsigned)((e.n + 255) / 256)), dim3(256), 0, s, e.ids, e.n, e.offsets, e.n_bags,
                           (int)e.vocab, w.bag, w.keys[0], w.perm[0]);
    if ((rc = (int)hipGetLastError())) return rc;
    CragSegArgs a = {};
    a.src = w.dp;
    a.n = e.n;
    a.dim = e.dim;
    a.vocab = (int)e.vocab;
    a.bag = w.bag;
    a.weights = e.weights;
    if (e.d_weights && e.n > 0) {
        const Shape sh = row_shape(e.dim, vec_of(e.dim, esz, {e.table}));
        a.lpr = sh.lpr;
        a.share = share_of(e.n, sh.lpr);
        a.n_share = (e.n + a.share - 1) / a.share;
        rc = e.dtype == CRAG_F32 ? launch_dweights<CRAG_F32>(a, sh, e.table, e.ids, e.d_weights, s)
                                 : launch_dweights<CRAG_BF16>(a, sh, e.table, e.ids, e.d_weights, s);
        if (rc) return rc;
    }
    if (!e.d_table) return 0;
    // rows of tokens that do not occur are zero
    const size_t bytes = (size_t)e.vocab * (size_t)e.dim * (size_t)esz;
    const size_t n16 = ((uintptr_t)e.d_table % 16) == 0 ? bytes / 16 : 0;
    if (n16 == 0 && bytes >= 16) return -3;  // refused by the caller
    const long long fill_blocks = std::max<long long>(1, std::min<long long>(8192, ((long long)n16 + 255) / 256));
    hipLaunchKernelGGL(k_fill_rows, dim3((unsigned)fill_blocks), dim3(256), 0, s, (u32x4_t*)e.d_table, (long long)n16,
                       (unsigned char*)e.d_table + n16 * 16, (int)(bytes - n16 * 16));
    if ((rc = (int)hipGetLastError())) return rc;
    if (e.n == 0) return 0;
    int cur = 0;
    if (e.n <= SORT_SMALL) {
        int P = 2;
        while (P < e.n) P <<= 1;
        hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(1024), sizeof(unsigned long long) * (size_t)P, s, w.keys[0], w.perm[0], (int)e.n, P);
    } else {
        const int tiles = (int)((e.n + SORT_TILE - 1) / SORT_TILE);
        for (int shift = 0; shift < 32 && (e.vocab >> shift) > 0; shift += 8) {
            hipLaunchKernelGGL(k_sort_count, dim3(tiles), dim3(256), 0, s, w.keys[cur], e.n, shift, tiles, w.hist);
            hipLaunchKernelGGL(k_sort_prefix, dim3(256), dim3(256), 0, s, w.hist, tiles, w.total);
            hipLaunchKernelGGL(k_sort_scatter, dim3(tiles), dim3(256), 0, s, w.keys[cur], w.perm[cur], e.n, shift, tiles, w.hist, w.total,
                               w.keys[cur ^ 1], w.perm[cur ^ 1]);
            cur ^= 1;
        }
    }
    if ((rc = (int)hipGetLastError())) return rc;
    const Shape sh = row_shape(e.dim, e.dim % 4 == 0 ? 4 : (e.dim % 2 == 0 ? 2 : 1));  // dp and partials: 256-byte aligned
    a.lpr = sh.lpr;
    a.share = share_of(e.n, sh.lpr);
    a.n_share = (e.n + a.share - 1) / a.share;
    a.keys = w.keys[cur];
    a.perm = w.perm[cur];
    a.partial = w.seg.partial;
    a.partial_seg = w.seg.partial_seg;
    a.partial_count = w.seg.partial_count;
    a.out = e.d_table;
    a.out_dtype = e.dtype;
    return launch_segsum<CRAG_F32, true>(a, sh, s);
}
