// Attention over the edges into a node (include/nbx.h "Block operators"): softmax of the edges' logits,
// dropout of the weights (drawn from the counter, never stored), weighted sum of the edges' values, and the
// backward pass.  Bound by HBM: every value is read once per direction; logits, weights and the CSR are a
// few words per edge and stay in LDS.
//   * list form: a block per (node, slice of the row) walks the node's list with a running maximum and sum;
//   * chunk form, for long lists: a block per 64 positions of the CSR, whatever nodes they belong to; a list
//     that crosses a chunk's border leaves partial sums with their own maximum, joined by a second launch.
// Backward: a block per few positions forms dvalues, the weights' gradient and, for lists that lie within
// the block, the softmax's own gradient; a second launch finishes the lists that cross blocks and the edges that
// no list entry names.
#include <algorithm>
#include <type_traits>

#include "nbx_internal.h"
#include "philox.h"
#include "typed_io.h"

namespace {

using namespace nbx;

constexpr int TILE = 64;      // positions whose weights are in LDS at once
constexpr int SA_MAXH = 64;
constexpr int AHEAD = 4;        // values of a thread that are on their way at once

// VW consecutive elements as loaded (RawV: waits only where it is used) and as fp32
template <typename T, int VW>
struct VecT {
    typedef T type __attribute__((ext_vector_type(VW), aligned(sizeof(T))));
};
template <typename T>
struct VecT<T, 1> {
    typedef T type;
};
template <typename T, int VW>
using RawV = typename VecT<T, VW>::type;
template <typename T, int VW>
__device__ __forceinline__ RawV<T, VW> loadr(const T* p) {
    return *reinterpret_cast<const RawV<T, VW>*>(p);
}
template <typename T, int VW>
__device__ __forceinline__ float lane_of(const RawV<T, VW>& r, int i) {
    if constexpr (VW == 1) return (float)r;
    else return (float)r[i];
}
template <typename T, int VW>
__device__ __forceinline__ void storev(T* p, const float (&v)[VW]) {
    if constexpr (VW == 1) {
        p[0] = (T)v[0];
    } else {
        RawV<T, VW> t;
#pragma unroll
        for (int i = 0; i < VW; ++i) t[i] = (T)v[i];
        *reinterpret_cast<RawV<T, VW>*>(p) = t;
    }
}

__device__ __forceinline__ float load_logit(const nbx_segment_attention_args& a, int64_t at) {
    return a.l_dtype == NBX_F32 ? ((const float*)a.logits)[at]
         : a.l_dtype == NBX_BF16 ? (float)((const bf16*)a.logits)[at] : (float)((const f16*)a.logits)[at];
}

__device__ __forceinline__ void store_dlogit(const nbx_segment_attention_args& a, int64_t at, float d) {
    if (a.l_dtype == NBX_F32) ((float*)a.dlogits)[at] = d;
    else if (a.l_dtype == NBX_BF16) ((bf16*)a.dlogits)[at] = (bf16)d;
    else ((f16*)a.dlogits)[at] = (f16)d;
}

// exp(l - m) with m the finite maximum (0 for a list that is all -inf)
__device__ __forceinline__ float weight_of(float l, float m) { return l == -INFINITY ? 0.f : __expf(l - m); }
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

struct SaPlan {
    int T, RV, EL, slices;    // threads, vectors per row, edges side by side, blocks per row
    int RB, spb, tile;        // join: vectors of a row per block; list form: slices per block, edges at a time
    int eb, TP, grp, entries; // backward: positions per block, threads that work, lanes of a head that shuffle,
                              // what they leave per position
    int chunked;
    int64_t nc;               // chunks (forward) or blocks (backward)
};

__device__ __forceinline__ void note_used(const nbx_segment_attention_args& a) {
    if (a.used && a.threshold && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        a.used[0] = a.rng[0];
        a.used[1] = a.rng[1];
    }
}

// The last v of [lo, V) with ptr[v] <= p (lo if there is none): a 64-way search by one wave.
__device__ __forceinline__ int64_t last_start(const int32_t* __restrict__ ptr, int64_t lo, int64_t V, int64_t p) {
    int64_t hi = V;
    while (hi - lo > 1) {
        const int64_t step = (hi - lo + 63) >> 6, at = lo + ((threadIdx.x & 63) + 1) * step;
        const uint64_t below = __ballot(at < hi && ptr[std::min(at, V)] <= p);
        lo += __popcll(below) * step;
        hi = std::min(hi, lo + step);
    }
    return lo;
}

// sV[i], i < cnt <= 64: the node whose list holds position p0 + i (the last v with ptr[v] <= p0 + i), or -1 in
// none.  One wave: a search for the first position, then the starts of the nodes after it are dropped on their
// positions and spread to the right.  A run of empty nodes is searched for its last one, so that at most two steps
// and a search go to each position, however many nodes start there (2^22 empty nodes between two lists, the backward
// pass: 24 ms walked 64 at a time, 0.02 ms searched).
__device__ __forceinline__ void nodes_of_positions(const int32_t* __restrict__ ptr, int64_t V, int64_t p0, int cnt,
                                                   int* sV) {
    const int lane = threadIdx.x & 63;
    const int64_t lo = last_start(ptr, 0, V, p0);
    sV[lane] = lane == 0 ? (int)lo : -1;
    __threadfence_block();
    for (int64_t v = lo + 1; v < V; v += 64) {
        const int64_t mine = v + lane;
        const int64_t at = mine < V ? ptr[mine] - p0 : cnt;
        if (at > 0 && at < cnt) atomicMax(&sV[at], (int)mine);
        if (__ballot(at >= cnt)) break;   // starts ascend: the later ones lie behind the block
        const int first = __builtin_amdgcn_readlane((int)at, 0);
        if (first == __builtin_amdgcn_readlane((int)at, 63)) {   // 64 nodes at one position
            v = last_start(ptr, v + 63, V, p0 + first);
            if (lane == 0 && first > 0 && first < cnt) atomicMax(&sV[first], (int)v);
            v -= 63;   // the loop's step goes on behind it
        }
    }
    __threadfence_block();
    int v = sV[lane];
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int left = __shfl_up(v, m, 64);
        if (lane >= m) v = std::max(v, left);
    }
    const int64_t p = p0 + lane;
    sV[lane] = V > 0 && lane < cnt && p >= ptr[v] && p < ptr[v + 1] ? v : -1;   // V = 0: ptr has one entry
}

// The lists that have positions in a block: sP[j] = first position of the j-th, sP[lists] = cnt; returns how
// many.  One wave, after nodes_of_positions.
__device__ __forceinline__ int lists_of_positions(const int* sV, int cnt, int* sP) {
    const int lane = threadIdx.x & 63;
    const bool first = lane < cnt && (lane == 0 || sV[lane] != sV[lane - 1]);
    const uint64_t m = __ballot(first);
    if (first) sP[__popcll(m & (((uint64_t)1 << lane) - 1))] = lane;
    const int n = __popcll(m);
    if (lane == 0) sP[n] = cnt;
    return n;
}

// max / sum over the 8 lanes of a (list, head)
__device__ __forceinline__ float max8(float x) {
#pragma unroll
    for (int m = 4; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
    return x;
}
__device__ __forceinline__ float sum8(float x) {
#pragma unroll
    for (int m = 4; m; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
}

// acc += w[i] row(i) over i = i0, i0 + step, .. < i1, AHEAD rows at a time; a weight of 0 reads nothing
template <typename T, int VW, typename W, typename R>
__device__ __forceinline__ void weighted_rows(float (&acc)[VW], int i0, int i1, int step, W&& weight, R&& row) {
    for (int i = i0; i < i1; i += AHEAD * step) {
        float w[AHEAD];
        RawV<T, VW> x[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = i + u * step;
            w[u] = k < i1 ? weight(k) : 0.f;
            if (w[u] != 0.f) x[u] = loadr<T, VW>(row(k));
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (w[u] != 0.f)
#pragma unroll
                for (int k = 0; k < VW; ++k) acc[k] = fmaf(w[u], lane_of<T, VW>(x[u], k), acc[k]);
    }
}

// Sum over the EL groups of RV threads (thread = el RV + f), left in group 0.
template <int VW>
__device__ __forceinline__ void join_groups(float (&acc)[VW], float* red, int RV, int EL) {
    const int t = threadIdx.x;
    __syncthreads();
    if (t < RV * EL)
#pragma unroll
        for (int i = 0; i < VW; ++i) red[t * VW + i] = acc[i];
    __syncthreads();
    if (t < RV)
        for (int g = 1; g < EL; ++g)
#pragma unroll
            for (int i = 0; i < VW; ++i) acc[i] += red[(g * RV + t) * VW + i];
}

// ======================================================================== forward, list form
// A block per node and `spb` slices of T vectors of its row.  A list of up to `tile` edges has its weights formed
// once for all slices, while the first slice's values are on their way; the next slice's are loaded before
// this one's result is stored.  640 nodes of 4 edges, rows of 49 x 8 x 16 fp32: 18 us, 80 MB at 4.4 TB/s.
template <typename T, int VW>
__global__ __launch_bounds__(256) void segment_attention_list_kernel(nbx_segment_attention_args a, SaPlan p, float keep) {
    extern __shared__ float lds[];
    const int H = a.H, t = threadIdx.x;
    float* sW = lds;                       // [tile][H] logits, then weights
    float* sM = sW + p.tile * H;           // [H] running maximum
    float* sR = sM + H;                    // [H] factor of what is summed so far
    float* sS = sR + H;                    // [H] running sum
    float* red = sS + H;                   // [T VW]
    int* sE = reinterpret_cast<int*>(red + p.T * VW);   // [tile]
    uint8_t* sK = reinterpret_cast<uint8_t*>(sE + p.tile);   // [tile][H]
    note_used(a);
    const DrawKey key = a.threshold ? draw_key(a.rng, a.call) : DrawKey{0, 0, 0, 0};
    const int64_t v = blockIdx.x;
    const int j0 = std::max(0, a.ptr[v]), j1 = (int)std::min<int64_t>(a.E, a.ptr[v + 1]);
    const int64_t RL = (int64_t)p.RV * VW;
    const int el = p.slices > 1 ? 0 : t / p.RV;
    const int s0 = blockIdx.y * p.spb, s1 = std::min(s0 + p.spb, p.slices);
    auto column = [&](int s) { return p.slices > 1 ? s * p.T + t : t - el * p.RV; };
    auto is_on = [&](int f) { return el < p.EL && f < p.RV; };
    auto value = [&](int i, int f) { return (const T*)a.values + (int64_t)sE[i] * RL + (int64_t)f * VW; };
    // the weights of positions [b, b + cnt) with the running maximum and sum; `meanwhile` runs once the edges
    // are known
    auto weigh = [&](int b, int cnt, auto&& meanwhile) {
        __syncthreads();
        for (int i = t; i < cnt; i += p.T) {
            const int e = a.eid[b + i];
            sE[i] = e >= 0 && e < a.E ? e : -1;
        }
        __syncthreads();
        meanwhile();
        for (int i = t; i < cnt * H; i += p.T) {
            const int e = sE[i / H];
            sW[i] = e < 0 ? -INFINITY : load_logit(a, (int64_t)e * H + i % H);
            sK[i] = !a.threshold || keep_one(key, (uint64_t)(int64_t)e * H + i % H, a.threshold);
        }
        __syncthreads();
        for (int h = t >> 3; h < H; h += p.T >> 3) {   // 8 lanes per head
            float m = -INFINITY, s = 0.f;
            for (int i = t & 7; i < cnt; i += 8) m = fmaxf(m, sW[i * H + h]);
            const float m0 = sM[h], s0 = sS[h], m1 = fmaxf(m0, max8(m));
            for (int i = t & 7; i < cnt; i += 8) {
                const float w = weight_of(sW[i * H + h], finite_max(m1));
                s += w;
                sW[i * H + h] = sK[i * H + h] ? w : 0.f;
            }
            s = sum8(s);
            if ((t & 7) == 0) {   // the 8 lanes have read what this replaces
                const float r = m0 == -INFINITY ? 0.f : __expf(m0 - m1);
                sR[h] = r;
                sM[h] = m1;
                sS[h] = s0 * r + s;
            }
        }
        __syncthreads();
    };
    auto finish = [&](float (&acc)[VW], int f, int head) {   // after a barrier that follows the sums
        if (is_on(f) && el == 0) {
            const float inv = keep / (sS[head] + 1e-16f);
#pragma unroll
            for (int k = 0; k < VW; ++k) acc[k] = sS[head] == 0.f ? 0.f : acc[k] * inv;
            storev<T, VW>((T*)a.out + v * RL + (int64_t)f * VW, acc);
        }
    };
    auto head_of = [&](int f) { return is_on(f) ? (f * VW / a.D) % H : 0; };
    if (j1 - j0 <= p.tile) {
        const int cnt = std::max(0, j1 - j0);
        RawV<T, VW> x[AHEAD];
        auto fetch = [&](int f) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int i = el + k * p.EL;
                if (is_on(f) && i < cnt && sE[i] >= 0) x[k] = loadr<T, VW>(value(i, f));
            }
        };
        if (t < H) {
            sM[t] = -INFINITY;
            sS[t] = 0.f;
        }
        weigh(j0, cnt, [&] { fetch(column(s0)); });
        for (int s = s0; s < s1; ++s) {
            const int f = column(s), head = head_of(f);
            float acc[VW] = {};
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = el + j * p.EL;
                const float w = is_on(f) && i < cnt ? sW[i * H + head] : 0.f;
                if (w != 0.f)
#pragma unroll
                    for (int k = 0; k < VW; ++k) acc[k] = fmaf(w, lane_of<T, VW>(x[j], k), acc[k]);
            }
            if (is_on(f) && cnt > AHEAD * p.EL)
                weighted_rows<T, VW>(acc, el + AHEAD * p.EL, cnt, p.EL, [&](int i) { return sW[i * H + head]; },
                                     [&](int i) { return value(i, f); });
            if (s + 1 < s1) fetch(column(s + 1));
            if (p.EL > 1) join_groups<VW>(acc, red, p.RV, p.EL);
            finish(acc, f, head);
        }
    } else {
        for (int s = s0; s < s1; ++s) {
            const int f = column(s), head = head_of(f);
            float acc[VW] = {};
            __syncthreads();
            if (t < H) {
                sM[t] = -INFINITY;
                sS[t] = 0.f;
            }
            for (int b = j0; b < j1; b += p.tile) {
                const int cnt = std::min(p.tile, j1 - b);
                weigh(b, cnt, [] {});
                const float r = sR[head];
#pragma unroll
                for (int k = 0; k < VW; ++k) acc[k] *= r;
                if (is_on(f))
                    weighted_rows<T, VW>(acc, el, cnt, p.EL, [&](int i) { return sW[i * H + head]; },
                                         [&](int i) { return value(i, f); });
            }
            if (p.EL > 1) join_groups<VW>(acc, red, p.RV, p.EL);
            else __syncthreads();
            finish(acc, f, head);
        }
    }
    if (a.stats && blockIdx.y == 0 && t < H) {
        a.stats[v * H + t] = finite_max(sM[t]);
        a.stats[(a.V + v) * H + t] = 1.0f / (sS[t] + 1e-16f);
    }
}

// ======================================================================== forward, chunk form
// 60000 edges of 8 x 64 bf16 to 96 nodes: 19 us (61 MB at 3.2 TB/s: the searches, logits and softmax come before
// the values) and 9.5 us for the join, whose longest list has 96 parts.
// partial sums of the lists that cross chunk c's borders: slot 2 c = the list that began before it, slot
// 2 c + 1 = the list that begins in it and goes on: acc [2 nc][RL] unnormalised, ms [2 nc][2][H] (max, sum)
template <typename T, int VW>
__global__ __launch_bounds__(256) void segment_attention_chunk_kernel(nbx_segment_attention_args a, SaPlan p, float keep,
                                                                      float* __restrict__ pacc, float* __restrict__ pms) {
    extern __shared__ float lds[];
    const int H = a.H, t = threadIdx.x;
    float* sW = lds;
    float* sM = sW + TILE * H;             // [TILE][H]: of the list that begins at the position
    float* sS = sM + TILE * H;
    float* red = sS + TILE * H;
    int* sE = reinterpret_cast<int*>(red + p.T * VW);
    int* sV = sE + TILE;
    int* sP = sV + TILE;                                   // [TILE + 1], then how many
    uint8_t* sK = reinterpret_cast<uint8_t*>(sP + TILE + 2);   // [TILE][H]
    note_used(a);
    const DrawKey key = a.threshold ? draw_key(a.rng, a.call) : DrawKey{0, 0, 0, 0};
    const int64_t c = blockIdx.x;
    const int p0 = (int)(c * TILE), cnt = (int)std::min<int64_t>(TILE, a.E - c * TILE);
    if (t < 64) {
        nodes_of_positions(a.ptr, a.V, p0, cnt, sV);
        __threadfence_block();
        const int n = lists_of_positions(sV, cnt, sP);
        if (t == 0) sP[TILE + 1] = n;
    } else if (t < 64 + cnt) {
        const int e = a.eid[p0 + t - 64];
        sE[t - 64] = e >= 0 && e < a.E ? e : -1;
    }
    __syncthreads();
    for (int i = t; i < cnt * H; i += p.T) {
        const int e = sE[i / H];
        sW[i] = e < 0 ? -INFINITY : load_logit(a, (int64_t)e * H + i % H);
        sK[i] = !a.threshold || keep_one(key, (uint64_t)(int64_t)e * H + i % H, a.threshold);
    }
    __syncthreads();
    const int lists = sP[TILE + 1];
    for (int k = t >> 3; k < lists * H; k += p.T >> 3) {   // 8 lanes per (list, head)
        const int i0 = sP[k / H], i1 = sP[k / H + 1], h = k % H;
        float m = -INFINITY, s = 0.f;
        for (int i = i0 + (t & 7); i < i1; i += 8) m = fmaxf(m, sW[i * H + h]);
        m = max8(m);
        for (int i = i0 + (t & 7); i < i1; i += 8) {
            const float w = weight_of(sW[i * H + h], finite_max(m));
            s += w;
            sW[i * H + h] = sK[i * H + h] ? w : 0.f;
        }
        s = sum8(s);
        if ((t & 7) == 0) {
            sM[i0 * H + h] = m;
            sS[i0 * H + h] = s;
        }
    }
    __syncthreads();
    const int el = p.slices > 1 ? 0 : t / p.RV;
    const int f = p.slices > 1 ? (int)blockIdx.y * p.T + t : t - el * p.RV;
    const bool on = el < p.EL && f < p.RV;
    const int head = on ? (f * VW / a.D) % H : 0;
    const int64_t RL = (int64_t)p.RV * VW;
    for (int j = 0; j < lists; ++j) {
        const int i0 = sP[j], i1 = sP[j + 1], v = sV[i0];
        if (v < 0) continue;
        float acc[VW] = {};
        if (on)
            weighted_rows<T, VW>(acc, i0 + el, i1, p.EL, [&](int i) { return sW[i * H + head]; },
                                 [&](int i) { return (const T*)a.values + (int64_t)sE[i] * RL + (int64_t)f * VW; });
        if (p.EL > 1) join_groups<VW>(acc, red, p.RV, p.EL);
        const bool before = a.ptr[v] < p0, after = std::min<int64_t>(a.E, a.ptr[v + 1]) > p0 + cnt;
        if (before || after) {
            const int64_t slot = 2 * c + (before ? 0 : 1);
            if (on && el == 0)
#pragma unroll
                for (int k = 0; k < VW; ++k) pacc[slot * RL + (int64_t)f * VW + k] = acc[k];
            if (blockIdx.y == 0 && t < H) {
                pms[(slot * 2) * H + t] = sM[i0 * H + t];
                pms[(slot * 2 + 1) * H + t] = sS[i0 * H + t];
            }
        } else {
            if (on && el == 0) {
                const float s = sS[i0 * H + head], inv = keep / (s + 1e-16f);
#pragma unroll
                for (int k = 0; k < VW; ++k) acc[k] = s == 0.f ? 0.f : acc[k] * inv;
                storev<T, VW>((T*)a.out + v * RL + (int64_t)f * VW, acc);
            }
            if (a.stats && blockIdx.y == 0 && t < H) {
                a.stats[(int64_t)v * H + t] = finite_max(sM[i0 * H + t]);
                a.stats[(a.V + v) * H + t] = 1.0f / (sS[i0 * H + t] + 1e-16f);
            }
        }
    }
}

// joins the partial sums of a list over its chunks, EL of them side by side; an empty list gives 0
template <typename T, int VW>
__global__ __launch_bounds__(256) void segment_attention_join_kernel(nbx_segment_attention_args a, SaPlan p, float keep,
                                                                     const float* __restrict__ pacc,
                                                                     const float* __restrict__ pms) {
    extern __shared__ float lds[];
    const int64_t v = blockIdx.x;
    const int t = threadIdx.x, H = a.H;
    const int j0 = std::max(0, a.ptr[v]), j1 = (int)std::min<int64_t>(a.E, a.ptr[v + 1]);
    const int64_t c0 = j0 / TILE, c1 = j1 > j0 ? (j1 - 1) / TILE : c0 - 1;
    if (c1 == c0) return;   // within one chunk: done there
    float* sR = lds;              // [TILE][H] factors of a tile of parts
    float* sQ = sR + TILE * H;    // [TILE][H] and their sums
    float* sM = sQ + TILE * H;    // [T] maxima, then [H] the list's
    float* sS = sM + p.T;         // [H]
    float* red = sS + H;          // [T VW]
    const int64_t RL = (int64_t)p.RV * VW;
    auto slot = [&](int64_t c) { return 2 * c + (j0 < c * TILE ? 0 : 1); };
    const int hs = p.T / H, h = t % H, r = t / H;   // threads per head
    float m = -INFINITY;
    if (r < hs)
        for (int64_t c = c0 + r; c <= c1; c += hs) m = fmaxf(m, pms[slot(c) * 2 * H + h]);
    sM[t] = m;
    __syncthreads();
    if (t < H) {
        for (int i = 1; i < hs; ++i) m = fmaxf(m, sM[i * H + t]);
        sM[t] = finite_max(m);
        sS[t] = 0.f;
    }
    const int el = t / p.RB, f = (int)blockIdx.y * p.RB + t - el * p.RB;
    const bool on = el < p.EL && f < p.RV;
    const int head = on ? (f * VW / a.D) % H : 0;
    float acc[VW] = {};
    for (int64_t b = c0; b <= c1; b += TILE) {
        const int cnt = (int)std::min<int64_t>(TILE, c1 + 1 - b);
        __syncthreads();
        for (int i = t; i < cnt * H; i += p.T) {
            const float* ms = pms + slot(b + i / H) * 2 * H + i % H;
            const float w = weight_of(ms[0], sM[i % H]);
            sR[i] = w;
            sQ[i] = w * ms[H];
        }
        __syncthreads();
        if (t < H) {
            float s = sS[t];
            for (int i = 0; i < cnt; ++i) s += sQ[i * H + t];
            sS[t] = s;
        }
        if (on)
            weighted_rows<float, VW>(acc, el, cnt, p.EL, [&](int i) { return sR[i * H + head]; },
                                     [&](int i) { return pacc + slot(b + i) * RL + (int64_t)f * VW; });
    }
    join_groups<VW>(acc, red, p.RB, p.EL);
    if (on && el == 0) {
        const float inv = keep / (sS[head] + 1e-16f);
#pragma unroll
        for (int k = 0; k < VW; ++k) acc[k] = sS[head] == 0.f ? 0.f : acc[k] * inv;
        storev<T, VW>((T*)a.out + v * RL + (int64_t)f * VW, acc);
    }
    if (a.stats && blockIdx.y == 0 && t < H) {
        a.stats[v * H + t] = sM[t];
        a.stats[(a.V + v) * H + t] = 1.0f / (sS[t] + 1e-16f);
    }
}

// ======================================================================== backward
// Positions [eb block, ..): dvalues = w dout[v], and with dp = keep/(1-p) <dout[v], values>_h the softmax's
// dl = a (dp - sum over the list of a dp).  A list that crosses the block's borders leaves its a, dp (per
// position) and its share of the sum: slot 2 block = the list that began before, 2 block + 1 = the one that
// goes on.  Threads: EL groups of RV, or (long rows) TP threads, a multiple of the H D / VW columns, over the
// row in steps of TP: either way a thread stays with one head.  2560 edges of 49 x 8 x 16 fp32: 35.5 us (145 MB at
// 4.1 TB/s) + 4 for the second launch; 60000 edges of 8 x 64 bf16: 30 us (123 MB at 4.1 TB/s) + 9 (the check of
// missing edges is about 1 of them; in it every block that a list crosses sums the shares of all the list's blocks).
template <typename T, int VW>
__global__ __launch_bounds__(1024) void segment_attention_bwd_kernel(nbx_segment_attention_args a, SaPlan p, float keep,
                                                                     float* __restrict__ wa, float* __restrict__ wd,
                                                                     float* __restrict__ share, int2* __restrict__ ends,
                                                                     int32_t* __restrict__ named) {
    extern __shared__ float lds[];
    const int H = a.H, t = threadIdx.x;
    float* sA = lds;                       // [eb][H] alpha
    float* sK = sA + p.eb * H;             // [eb][H] keep / (1 - p) or 0
    float* sD = sK + p.eb * H;             // [eb][H] dp
    float* red = sD + p.eb * H;            // [eb][entries]: sums over grp lanes
    int* sE = reinterpret_cast<int*>(red + p.eb * p.entries);   // [64]
    int* sV = sE + 64;
    int* sP = sV + 64;                     // [64 + 1], then how many
    const DrawKey key = a.threshold ? draw_key(a.rng, a.call) : DrawKey{0, 0, 0, 0};
    const int64_t p0 = blockIdx.x * (int64_t)p.eb;
    const int cnt = (int)std::min<int64_t>(p.eb, a.E - p0);
    if (t < 64) {
        nodes_of_positions(a.ptr, a.V, p0, cnt, sV);
        __threadfence_block();
        const int n = lists_of_positions(sV, cnt, sP);
        if (t == 0) sP[65] = n;
    } else if (t < 64 + cnt) {
        const int e = a.eid[p0 + t - 64];
        sE[t - 64] = e >= 0 && e < a.E ? e : -1;
        if (e >= 0 && e < a.E) named[e] = (int32_t)(p0 + t - 64);
    }
    __syncthreads();
    for (int i = t; i < cnt * H; i += p.T) {
        const int e = sE[i / H], h = i % H;
        const int64_t v = sV[i / H];   // -1: in no list, its gradients are 0
        float al = 0.f, k = 0.f;
        if (e >= 0 && v < 0 && a.dlogits) store_dlogit(a, (int64_t)e * H + h, 0.f);
        if (e >= 0 && v >= 0) {
            al = weight_of(load_logit(a, (int64_t)e * H + h), a.stats[v * H + h]) * a.stats[(a.V + v) * H + h];
            k = !a.threshold || keep_one(key, (uint64_t)(int64_t)e * H + h, a.threshold) ? keep : 0.f;
        }
        sA[i] = al;
        sK[i] = k;
    }
    __syncthreads();
    const bool wide = p.RV > p.T;          // one edge at a time, several vectors a thread
    const int cols = H * a.D / VW, el = wide ? 0 : t / p.RV, f0 = wide ? t : t - el * p.RV;
    const bool on = wide ? t < p.TP : el < p.EL;
    const int head = on ? (f0 * VW / a.D) % H : 0;
    const int64_t RL = (int64_t)p.RV * VW;
    // items of a thread: AHEAD of its positions (one vector each), or AHEAD vectors of one position
    const int nf = wide ? (p.RV + p.TP - 1) / p.TP : 1, items = (wide ? cnt : (cnt + p.EL - 1) / p.EL) * nf;
    float s = 0.f;
    for (int q = 0; q < items; q += AHEAD) {
        RawV<T, VW> d[AHEAD], x[AHEAD];
        float w[AHEAD];
        int at[AHEAD], pos[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = q + u, i = wide ? k / nf : k * p.EL + el, f = wide ? f0 + k % nf * p.TP : f0;
            const bool live = on && k < items && i < cnt && f < p.RV && sE[i] >= 0;
            pos[u] = i;
            at[u] = live ? f : -1;
            w[u] = live ? sA[i * H + head] * sK[i * H + head] : 0.f;
            if (w[u] != 0.f) {
                d[u] = loadr<T, VW>((const T*)a.dout + (int64_t)sV[i] * RL + (int64_t)f * VW);
                if (a.dlogits) x[u] = loadr<T, VW>((const T*)a.values + (int64_t)sE[i] * RL + (int64_t)f * VW);
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            float g[VW];
#pragma unroll
            for (int k = 0; k < VW; ++k) {
                const float dk = lane_of<T, VW>(d[u], k);
                g[k] = w[u] == 0.f ? 0.f : dk * w[u];
                if (w[u] != 0.f && a.dlogits) s = fmaf(dk, lane_of<T, VW>(x[u], k), s);
            }
            if (a.dvalues && at[u] >= 0)
                storev<T, VW>((T*)a.dvalues + (int64_t)sE[pos[u]] * RL + (int64_t)at[u] * VW, g);
            if (q + u < items && (!wide || (q + u) % nf == nf - 1)) {   // a position of this thread is complete
                if (a.dlogits) {
                    for (int m = p.grp >> 1; m; m >>= 1) s += __shfl_xor(s, m, 64);
                    if (on && t % p.grp == 0 && pos[u] < cnt) red[pos[u] * p.entries + (wide ? t : f0) / p.grp] = s;
                }
                s = 0.f;
            }
        }
    }
    if (!a.dlogits) return;
    if (t == 0) ends[blockIdx.x] = make_int2(sV[0], sV[cnt - 1]);
    __syncthreads();
    // red: a position's entries are rows of `per` per head
    const int per = a.D / VW / p.grp, rows = p.entries / (cols / p.grp);
    for (int k = t; k < cnt * H; k += p.T) {
        const float* r = red + k / H * p.entries + k % H * per;
        float sum = 0.f;
        for (int j = 0; j < rows; ++j)
            for (int i = 0; i < per; ++i) sum += r[j * (cols / p.grp) + i];
        sD[k] = sK[k] == 0.f ? 0.f : sK[k] * sum;
    }
    __syncthreads();
    const int lists = sP[65];
    for (int k = t >> 3; k < lists * H; k += p.T >> 3) {   // 8 lanes per (list, head)
        const int i0 = sP[k / H], i1 = sP[k / H + 1], h = k % H, v = sV[i0];
        float d = 0.f;
        for (int i = i0 + (t & 7); i < i1; i += 8) d += sA[i * H + h] * sD[i * H + h];
        d = sum8(d);
        if (v < 0) continue;
        const bool before = a.ptr[v] < p0, after = std::min<int64_t>(a.E, a.ptr[v + 1]) > p0 + cnt;
        if ((before || after) && (t & 7) == 0) share[(2 * (int64_t)blockIdx.x + (before ? 0 : 1)) * H + h] = d;
        for (int i = i0 + (t & 7); i < i1; i += 8) {
            const float al = sA[i * H + h], dp = sD[i * H + h];
            if (before || after) {
                wa[(p0 + i) * H + h] = al;
                wd[(p0 + i) * H + h] = dp;
            } else if (sE[i] >= 0) {
                store_dlogit(a, (int64_t)sE[i] * H + h, al == 0.f ? 0.f : al * (dp - d));
            }
        }
    }
}

// Finishes the lists that cross the block's borders: at most one that began before it and one that goes on.  And
// the edges [p0, p0 + cnt) that no entry of eid names get gradients of 0: edge e is named iff eid[named[e]] = e,
// whatever named[e] held before, so `named` needs no clearing.
__global__ __launch_bounds__(256) void segment_attention_finish_kernel(nbx_segment_attention_args a, SaPlan p,
                                                                       const float* __restrict__ wa,
                                                                       const float* __restrict__ wd,
                                                                       const float* __restrict__ share,
                                                                       const int2* __restrict__ ends,
                                                                       const int32_t* __restrict__ named) {
    __shared__ float red[256];
    __shared__ uint64_t sMissing;
    const int t = threadIdx.x, H = a.H;
    const int64_t p0 = blockIdx.x * (int64_t)p.eb;
    const int cnt = (int)std::min<int64_t>(p.eb, a.E - p0);
    int2 ends_here = make_int2(-1, -1);   // the nodes of the block's first and last position
    if (a.dlogits) ends_here = ends[blockIdx.x];
    if (t < 64) {
        bool missing = false;
        if (t < cnt) {
            const int32_t at = named[p0 + t];
            missing = at < 0 || at >= a.E || a.eid[at] != p0 + t;
        }
        const uint64_t m = __ballot(missing);
        if (t == 0) sMissing = m;
    }
    __syncthreads();
    const int64_t halves = (int64_t)a.K * H * a.D * (a.v_dtype == NBX_F32 ? 2 : 1);   // 16-bit units of a row
    for (uint64_t m = sMissing; m; m &= m - 1) {
        const int64_t e = p0 + __ffsll((unsigned long long)m) - 1;
        if (a.dvalues)
            for (int64_t i = t; i < halves; i += 256) ((uint16_t*)a.dvalues)[e * halves + i] = 0;
        if (a.dlogits && t < H) store_dlogit(a, e * H + t, 0.f);
    }
    if (!a.dlogits) return;
    const int hs = 256 / H, h = t % H, r = t / H;
    for (int side = 0; side < 2; ++side) {
        const int v = side ? ends_here.y : ends_here.x;
        if (v < 0 || (side && v == ends_here.x)) continue;
        const int64_t q0 = std::max(0, a.ptr[v]), q1 = std::min<int64_t>(a.E, a.ptr[v + 1]);
        if (q0 >= p0 && q1 <= p0 + cnt) continue;
        const int64_t b0 = q0 / p.eb, b1 = (q1 - 1) / p.eb;
        float s = 0.f;
        if (r < hs)
#pragma unroll 4
            for (int64_t b = b0 + r; b <= b1; b += hs) s += share[(2 * b + (q0 < b * p.eb ? 0 : 1)) * H + h];
        __syncthreads();
        red[t] = s;
        __syncthreads();
        float delta = 0.f;
        for (int i = 0; i < hs; ++i) delta += red[i * H + h];
        const int64_t from = std::max(q0, p0), to = std::min(q1, p0 + cnt);
        if (r < hs)
            for (int64_t j = from + r; j < to; j += hs) {
                const int e = a.eid[j];
                if (e < 0 || e >= a.E) continue;
                const float al = wa[j * H + h];
                store_dlogit(a, (int64_t)e * H + h, al == 0.f ? 0.f : al * (wd[j * H + h] - delta));
            }
    }
}

// ======================================================================== host
bool dtype_ok(int32_t d) { return d == NBX_F32 || d == NBX_BF16 || d == NBX_F16; }

int vector_width(const nbx_segment_attention_args& a) {
    if (a.v_dtype != NBX_F32 && a.D % 8 == 0) return 8;
    return a.D % 4 == 0 ? 4 : 1;
}

int sa_check(const nbx_segment_attention_args* a, const char* who) {
    NBX_CHECK_ARG(a, "%s: null arguments", who);
    const int64_t lim = (int64_t)1 << 31;
    // a list is walked in steps of up to 4 TILE positions held in 32 bits: the step past the last has to fit
    NBX_CHECK_ARG(a->V >= 0 && a->V < lim - 1 && a->E >= 0 && a->E < lim - 4 * TILE && a->K >= 1 && a->H >= 1 && a->D >= 1,
                  "%s: bad sizes", who);
    NBX_CHECK_ARG(dtype_ok(a->v_dtype) && (a->l_dtype == a->v_dtype || a->l_dtype == NBX_F32),
                  "%s: l_dtype must be fp32 or v_dtype", who);
    NBX_CHECK_ARG(a->H <= SA_MAXH && a->D <= 4096 && (int64_t)a->H * a->D <= (a->D % 4 == 0 ? 4096 : 1024),
                  "%s: need H <= %d, H D <= 4096 (1024 if D %% 4)", who, SA_MAXH);
    NBX_CHECK_ARG(a->K < (1 << 20) && a->K * a->H * a->D < (1 << 20), "%s: need K H D < 2^20", who);
    NBX_CHECK_ARG(a->V < (1 << 24), "%s: too many nodes", who);   // a launch's threads along x fit 32 bits
    NBX_CHECK_ARG(a->threshold < 65536 && (!a->threshold || a->rng), "%s: need threshold < 65536, and rng for a drop rate",
                  who);
    return NBX_OK;
}

SaPlan forward_plan(const nbx_segment_attention_args& a) {
    SaPlan p = {};
    const int VW = vector_width(a);
    p.T = 256;
    p.RV = (int)(a.K * a.H * a.D / VW);
    p.EL = p.RV <= p.T ? p.T / p.RV : 1;
    p.slices = p.RV <= p.T ? 1 : (int)ceil_div(p.RV, p.T);
    // The lists' lengths are on the device.  E a multiple of V is taken for lists of one length (a fully connected
    // graph): the list form up to 128 edges (K 1, 8 heads of 16, fp32, both passes: 4096 x 7 37 us against 53 in
    // chunks, 2048 x 15 31 / 43, 1040 x 64 40 / 43, 516 x 128 43 / 47).  Otherwise chunks, which do not wait for the
    // longest list (ragged lists, 60001 edges to 3000 nodes: 61 us, to 1000: 52; 20001 to 2000: 56), but for small
    // graphs, where the list form's single launch counts.  It is a guess: ragged lists whose E happens to be a multiple
    // of V run the list form too, and wait for the longest list (60000 edges to 3000 nodes: 107 us, to 1000: 157; 20000
    // to 2000: 60).
    p.chunked = a.V && a.E % a.V == 0 ? a.E > 128 * a.V : a.E > 1024;
    // edges whose weights a list's block forms at once: 256 for long lists (60000 edges to 1000 nodes in list form:
    // 127 us against 151 at 64), 64 where lists are short or heads many, for the LDS
    p.tile = a.E <= 8 * a.V || a.H > 32 ? TILE : 4 * TILE;
    // about 1024 blocks or more: 640 nodes of 7 slices take 24.4 us at one slice per block, 20.3 at two, 18.1 at
    // four, 19.2 at seven
    p.spb = (int)ceil_div(p.slices, std::min<int64_t>(p.slices, std::max<int64_t>(1, ceil_div(1024, std::max<int64_t>(1, a.V)))));
    p.nc = ceil_div(a.E, TILE);
    return p;
}

SaPlan backward_plan(const nbx_segment_attention_args& a) {
    SaPlan p = {};
    const int VW = vector_width(a), cols = a.H * a.D / VW;
    p.T = std::max(256, (int)ceil_div(cols, 64) * 64);
    p.RV = (int)(a.K * a.H * a.D / VW);
    p.EL = p.RV <= p.T ? std::min(p.T / p.RV, TILE) : 1;
    p.TP = p.RV <= p.T ? p.RV * p.EL : p.T / cols * cols;
    const int g = a.D / VW;
    p.grp = g <= 64 && (g & (g - 1)) == 0 ? g : 1;
    p.entries = std::min(p.RV, p.TP) / p.grp;
    // positions per block: enough blocks for the chip first, then few (each has its searches and sums), within
    // 48 KB of LDS: 60000 edges of 8 x 64 bf16 take 49 us at 16, 42 at 32, 39 at 64; long rows (2560 edges of 49 x 8
    // x 16 fp32) 40 us at 2, 38 at 4, 48 at 8, 77 at 16
    p.eb = p.RV <= p.T ? TILE : 4;
    while (p.eb > 4 && (a.E < 768 * (int64_t)p.eb || p.eb * (p.entries + 3 * a.H) > 12288)) p.eb /= 2;
    p.eb = std::max(p.eb, std::min(p.EL, TILE));
    // lists of one length (a fully connected graph): whole lists per block, so that none crosses
    const int64_t d = a.V && a.E % a.V == 0 ? a.E / a.V : 0;
    if (d >= 1 && d <= p.eb) p.eb = (int)(p.eb / d * d);
    else if (d > p.eb && d <= std::min(2 * p.eb, TILE) && d * (p.entries + 3 * a.H) <= 12288) p.eb = (int)d;
    p.nc = ceil_div(a.E, p.eb);
    return p;
}

// f(T{}, std::integral_constant<int, VW>{})
template <typename F>
int with_values(const nbx_segment_attention_args& a, F&& f) {
    const int VW = vector_width(a);
    auto pick = [&](auto t) -> int {
        if constexpr (sizeof(t) == 2)
            if (VW == 8) return f(t, std::integral_constant<int, 8>{});
        if (VW == 4) return f(t, std::integral_constant<int, 4>{});
        return f(t, std::integral_constant<int, 1>{});
    };
    if (a.v_dtype == NBX_F32) return pick(float{});
    if (a.v_dtype == NBX_BF16) return pick(bf16{});
    return pick(f16{});
}

size_t workspace_need(const nbx_segment_attention_args& a, bool backward) {
    if (backward) {
        const int64_t nc = backward_plan(a).nc;
        return (size_t)((a.dlogits ? 2 * ((a.E + nc) * a.H + nc) : 0) + a.E) * sizeof(float);
    }
    const SaPlan p = forward_plan(a);
    return p.chunked ? (size_t)2 * p.nc * (a.K * a.H * a.D + 2 * a.H) * sizeof(float) : 0;
}

}  // namespace

// ======================================================================== C ABI (include/nbx.h)
extern "C" int nbx_segment_attention_workspace_bytes(const nbx_segment_attention_args* a, int32_t backward,
                                                     size_t* bytes) {
    if (int rc = sa_check(a, "nbx_segment_attention_workspace_bytes")) return rc;
    NBX_CHECK_ARG(bytes, "nbx_segment_attention_workspace_bytes: null result");
    *bytes = workspace_need(*a, backward != 0);
    return NBX_OK;
}

extern "C" int nbx_segment_attention(const nbx_segment_attention_args* a, void* stream) {
    if (int rc = sa_check(a, "nbx_segment_attention")) return rc;
    if (a->V == 0) return NBX_OK;
    NBX_CHECK_ARG(a->ptr && a->out && (a->E == 0 || (a->eid && a->values && a->logits)),
                  "nbx_segment_attention: null operand");
    const size_t need = workspace_need(*a, false);
    if (need && !(a->workspace && a->workspace_bytes >= need)) {
        set_error("nbx_segment_attention: workspace too small");
        return NBX_E_WORKSPACE;
    }
    const SaPlan p = forward_plan(*a);
    NBX_CHECK_ARG(!p.chunked || p.nc * p.T < ((int64_t)1 << 32), "nbx_segment_attention: too many edges");
    hipStream_t st = (hipStream_t)stream;
    const float keep = keep_scale(a->threshold);
    return with_values(*a, [&](auto t, auto vw) -> int {
        using T = decltype(t);
        constexpr int VW = decltype(vw)::value;
        if (!p.chunked) {
            const size_t lds = (size_t)(p.tile * a->H + 3 * a->H + p.T * VW + p.tile) * 4 + p.tile * a->H;
            hipLaunchKernelGGL((segment_attention_list_kernel<T, VW>), dim3((unsigned)a->V, (unsigned)ceil_div(p.slices, p.spb)),
                               dim3(p.T), lds, st, *a, p, keep);
            NBX_LAUNCH_CHECK("segment_attention_list");
            return NBX_OK;
        }
        float* pacc = (float*)a->workspace;
        float* pms = pacc + 2 * p.nc * a->K * a->H * a->D;
        const size_t lds = (size_t)(3 * TILE * a->H + p.T * VW + 3 * TILE + 2) * 4 + TILE * a->H;   // <= 62 KB
        if (p.nc) {
            hipLaunchKernelGGL((segment_attention_chunk_kernel<T, VW>), dim3((unsigned)p.nc, (unsigned)p.slices), dim3(p.T),
                               lds, st, *a, p, keep, pacc, pms);
            NBX_LAUNCH_CHECK("segment_attention_chunk");
        }
        SaPlan j = p;   // sixteen vectors of a row per block, so that many parts are read side by side
        j.RB = std::min(p.RV, 16);
        j.EL = 256 / j.RB;
        j.slices = (int)ceil_div(p.RV, j.RB);
        const size_t jlds = (size_t)(2 * TILE * a->H + p.T + a->H + p.T * VW) * 4;
        hipLaunchKernelGGL((segment_attention_join_kernel<T, VW>), dim3((unsigned)a->V, (unsigned)j.slices), dim3(p.T),
                           jlds, st, *a, j, keep, pacc, pms);
        NBX_LAUNCH_CHECK("segment_attention_join");
        return NBX_OK;
    });
}

extern "C" int nbx_segment_attention_backward(const nbx_segment_attention_args* a, void* stream) {
    if (int rc = sa_check(a, "nbx_segment_attention_backward")) return rc;
    if (a->E == 0 || (!a->dvalues && !a->dlogits)) return NBX_OK;   // without a node the gradients are 0
    NBX_CHECK_ARG(a->ptr && a->eid && a->values && a->logits && (a->V == 0 || (a->stats && a->dout)),
                  "nbx_segment_attention_backward: null operand");
    const size_t need = workspace_need(*a, true);
    if (need && !(a->workspace && a->workspace_bytes >= need)) {
        set_error("nbx_segment_attention_backward: workspace too small");
        return NBX_E_WORKSPACE;
    }
    const SaPlan p = backward_plan(*a);
    NBX_CHECK_ARG(p.nc * p.T < ((int64_t)1 << 32), "nbx_segment_attention_backward: too many edges");
    hipStream_t st = (hipStream_t)stream;
    const float keep = keep_scale(a->threshold);
    int2* ends = (int2*)a->workspace;   // ends, wa, wd and share only for dlogits
    float* wa = (float*)(ends + p.nc);
    float* wd = wa + a->E * a->H;
    float* share = wd + a->E * a->H;
    int32_t* named = a->dlogits ? (int32_t*)(share + 2 * p.nc * a->H) : (int32_t*)a->workspace;
    if (int rc = with_values(*a, [&](auto t, auto vw) -> int {
            using T = decltype(t);
            constexpr int VW = decltype(vw)::value;
            const size_t lds = (size_t)(3 * p.eb * a->H + p.eb * p.entries + 196) * 4;
            hipLaunchKernelGGL((segment_attention_bwd_kernel<T, VW>), dim3((unsigned)p.nc), dim3(p.T), lds, st, *a, p, keep,
                               wa, wd, share, ends, named);
            NBX_LAUNCH_CHECK("segment_attention_bwd");
            return NBX_OK;
        }))
        return rc;
    hipLaunchKernelGGL(segment_attention_finish_kernel, dim3((unsigned)p.nc), dim3(256), 0, st, *a, p, wa, wd, share, ends,
                       named);
    NBX_LAUNCH_CHECK("segment_attention_finish");
    return NBX_OK;
}
