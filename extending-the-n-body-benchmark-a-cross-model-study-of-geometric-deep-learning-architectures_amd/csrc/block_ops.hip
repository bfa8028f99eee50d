// Block operators (include/nbx.h "Block operators"): what surrounds the products of a training block —
//   * dropout whose mask is never stored (drawn again from the counter in the backward pass);
//   * the residual add with the norms before and after it, the gate (layer scale) and dropout;
//   * the same with EquiformerV2's spherical-harmonics norm.
// All three are bound by HBM: each element is read and written once per direction, everything else
// (statistics, draws, gate) happens in registers between the two.  A row lives in the registers of the 16
// or 64 lanes or of the block that owns it, eight consecutive columns per lane, so the norm's two passes
// (mean, then squares around it) cost no second read.  Column sums (parameter gradients) stay in registers
// over a block's rows, then one partial row per block is summed by a second launch in a fixed order.
#include <algorithm>
#include <type_traits>

#include "nbx_internal.h"
#include "philox.h"
#include "typed_io.h"

namespace {

using namespace nbx;

bool dtype_ok(int32_t d) { return d == NBX_F32 || d == NBX_BF16 || d == NBX_F16; }

// a launch's threads along x fit 32 bits
bool grid_ok(int64_t blocks, int threads) { return blocks * threads < ((int64_t)1 << 32); }

// f(T{}) with T the storage type of a dtype code
template <typename F>
int with_type(int32_t d, F&& f) {
    if (d == NBX_F32) return f(float{});
    if (d == NBX_BF16) return f(bf16{});
    return f(f16{});
}

__device__ __forceinline__ void note_used(int64_t* used, const int64_t* rng) {
    if (used && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        used[0] = rng[0];
        used[1] = rng[1];
    }
}

// ======================================================================== dropout
// Flat form: thread t owns elements 8 t .. 8 t + 7, which are exactly one Philox block's draws (16 bits a draw:
// with 32 the generator's 20 wide multiplies per four elements would take longer than 16-bit elements' way
// through HBM).  33.5M bf16 elements: 24 us, 134 MB at 5.5 TB/s (partly from the last-level cache).
template <typename T>
__global__ __launch_bounds__(256) void dropout_flat_kernel(int64_t total, uint32_t threshold, float scale,
                                                           const int64_t* __restrict__ rng, uint32_t call,
                                                           int64_t* __restrict__ used, const T* __restrict__ X,
                                                           T* __restrict__ Y) {
    note_used(used, rng);
    const int64_t q = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (8 * q >= total) return;
    const int n = (int)std::min<int64_t>(8, total - 8 * q);
    float v[8];
    load8n(X + 8 * q, n, v);
    const Keep8 m = keep_eight(draw_key(rng, call), (uint64_t)q, threshold);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = m.k[i] ? v[i] * scale : 0.f;
    store8n(Y + 8 * q, n, v);
}

// Row form (entries of S C elements sharing draws): a block takes 256 chunks of eight elements, of one
// entry or of several.  CHANNEL keeps the mask of the block's channels as bits in LDS, one Philox block for
// eight channels, shared by the S rows: all of a short row's, or the window of 2048 channels (wrapping at C)
// that a part of a long row touches.  8M fp32 elements: 13.5 us, 64 MB at 4.8 TB/s.
constexpr int CHANNEL_WINDOW = 2048 / 8 + 2;

template <typename T, bool CHANNEL>
__global__ __launch_bounds__(256) void dropout_rows_kernel(int64_t n, int64_t RS, int64_t C, int64_t group, int cpr,
                                                           int rpb, int64_t segs, uint32_t threshold, float scale,
                                                           const int64_t* __restrict__ rng, uint32_t call,
                                                           int64_t* __restrict__ used, const T* __restrict__ X,
                                                           T* __restrict__ Y) {
    __shared__ uint8_t mask[CHANNEL ? CHANNEL_WINDOW : 1];
    note_used(used, rng);
    const DrawKey key = draw_key(rng, call);
    const int64_t row0 = blockIdx.x / segs * rpb, seg = blockIdx.x % segs;
    const int64_t Cq = (C + 7) >> 3;
    const int64_t first = rpb > 1 ? 0 : seg * 2048 % C >> 3;             // the window's first byte
    const int per = (int)(Cq < CHANNEL_WINDOW ? Cq : CHANNEL_WINDOW);   // bytes per entry
    if (CHANNEL) {
        const int rows = (int)std::min<int64_t>(rpb, n - row0);
        for (int k = threadIdx.x; k < rows * per; k += 256) {
            const int64_t q = first + k % per;
            mask[k] = (uint8_t)keep_bits(key, (uint64_t)((row0 + k / per) * Cq + (q < Cq ? q : q - Cq)), threshold);
        }
        __syncthreads();
    }
    const int lr = rpb > 1 ? (int)threadIdx.x / cpr : 0;
    const int64_t row = row0 + lr, f0 = 8 * (rpb > 1 ? (int64_t)(threadIdx.x - lr * cpr) : seg * 256 + threadIdx.x);
    if (lr >= rpb || row >= n || f0 >= RS) return;
    const int cnt = (int)std::min<int64_t>(8, RS - f0);
    const int64_t at = row * RS + f0;
    float v[8];
    load8n(X + at, cnt, v);
    if (CHANNEL) {
        const uint8_t* mk = mask + lr * per;
        int64_t c = f0 % C;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t q = (c >> 3) - first;
            v[i] = (mk[q < 0 ? q + Cq : q] >> (c & 7) & 1) ? v[i] * scale : 0.f;
            c = c + 1 == C ? 0 : c + 1;
        }
    } else {
        const bool keep = keep_one(key, (uint64_t)(row / group), threshold);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = keep ? v[i] * scale : 0.f;
    }
    store8n(Y + at, cnt, v);
}

// ======================================================================== residual add, norms, gate
// Sum over the threads of a row: 16 or 64 lanes, or (W = 0) the whole block through LDS.  `slot` alternates
// over four places so that one barrier per sum is enough.
template <int W>
__device__ __forceinline__ float row_sum(float x, float (*red)[16], int& slot) {
    if constexpr (W != 0) {
        return lanes_sum<W>(x);
    } else {
        x = lanes_sum<64>(x);
        float* r = red[slot];
        slot = (slot + 1) & 3;
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = x;
        __syncthreads();
        float s = 0.f;
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += r[i];
        return s;
    }
}

// mean (0 for the RMS norm) and 1/sqrt(mean square around it + eps) of the row's n of eight columns here
template <int W>
__device__ __forceinline__ void row_stats(const float (&v)[8], int n, int C, int rms, float eps, float& mu, float& rs,
                                          float (*red)[16], int& slot) {
    mu = 0.f;
    if (!rms) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];   // columns past the row are 0
        mu = row_sum<W>(s, red, slot) / (float)C;
    }
    float q = 0.f;
    if (n == 8 || rms) {   // columns past the row are 0
#pragma unroll
        for (int i = 0; i < 8; ++i) q += (v[i] - mu) * (v[i] - mu);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = i < n ? v[i] - mu : 0.f;
            q += d * d;
        }
    }
    rs = 1.0f / sqrtf(row_sum<W>(q, red, slot) / (float)C + eps);
}

struct Draws {
    DrawKey key;
    uint32_t threshold;
    int64_t group, Cq;
    float scale;
};

// whether a row's eight columns at 8 lane are kept
__device__ __forceinline__ Keep8 row_keep(const Draws& d, int64_t row, int lane) {
    if (d.threshold == 0) return keep_all(true);
    if (d.group) return keep_all(keep_one(d.key, (uint64_t)(row / d.group), d.threshold));
    return keep_eight(d.key, (uint64_t)(row * d.Cq + lane), d.threshold);
}

// Forward: one row per 16 / 64 lanes or per block; the draws are formed while the row is on its way.  16384 rows
// of 2048 bf16 columns with both norms, gate and draws: 64 us, 268 MB at 4.2 TB/s (a copy: 4.8).  Several rows
// per block with the next one prefetched take 70 us: twice the registers, half the waves.
template <typename TX, typename TY, int W>
__global__ __launch_bounds__(W ? 256 : 1024) void residual_norm_kernel(nbx_residual_norm_args a, float keep) {
    __shared__ float red[4][16];
    int slot = 0;
    if (a.threshold) note_used(a.used, a.rng);
    const int lane = W ? (int)threadIdx.x % (W ? W : 1) : (int)threadIdx.x;
    const int64_t r = W ? blockIdx.x * (int64_t)(256 / (W ? W : 1)) + threadIdx.x / (W ? W : 1) : blockIdx.x;
    if (r >= a.rows) return;   // W = 0: never (one block per row); else whole lane groups
    const int C = (int)a.C, c0 = 8 * lane, n = std::max(0, std::min(8, C - c0));
    Draws d = {{0, 0, 0, 0}, a.threshold, a.group, (a.C + 7) >> 3, keep};
    if (a.threshold) d.key = draw_key(a.rng, a.call);
    Raw8<TX> rx;
    Raw8<TY> ry;
    fetch8n((const TX*)a.x + r * a.ldx + c0, n, rx);
    fetch8n((const TY*)a.y + r * a.ldy + c0, n, ry);
    const Keep8 m = row_keep(d, r, lane);   // while the rows are on their way
    float x[8], u[8], w[8], b[8];
    unpack8(rx, x);
    unpack8(ry, u);
    if (a.post_w) {
        float mu, rs;
        row_stats<W>(u, n, C, a.norm, a.eps, mu, rs, red, slot);
        load8p(a.post_w, a.param_dtype, c0, n, w);
        if (a.post_b) load8p(a.post_b, a.param_dtype, c0, n, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = (u[i] - mu) * rs * w[i] + (a.post_b ? b[i] : 0.f);
        if (a.stats && lane == 0) {
            a.stats[r] = mu;
            a.stats[a.rows + r] = rs;
        }
    }
    if (a.gate) {
        load8p(a.gate, a.param_dtype, (a.gate_groups == a.rows ? r : r / (a.rows / a.gate_groups)) * a.C + c0, n, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] *= w[i];
    }
    const float s = a.scale * keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(s, m.k[i] ? u[i] : 0.f, x[i]);
    store8n((TX*)a.h + r * a.C + c0, n, x);
    if (a.pre_w) {
        // z is the norm of the sum before h is rounded to its type: one rounding per result
        float mu, rs;
        row_stats<W>(x, n, C, a.norm, a.eps, mu, rs, red, slot);
        load8p(a.pre_w, a.param_dtype, c0, n, w);
        if (a.pre_b) load8p(a.pre_b, a.param_dtype, c0, n, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (x[i] - mu) * rs * w[i] + (a.pre_b ? b[i] : 0.f);
        store8n((TY*)a.z + r * a.C + c0, n, x);
        if (a.stats && lane == 0) {
            a.stats[2 * a.rows + r] = mu;
            a.stats[3 * a.rows + r] = rs;
        }
    }
}

// Which rows a block of the backward pass owns.  A block has `rpb` row slots: 16 or 64 lanes, or (W = 0) nw
// waves each.  ALIGNED: rows [g rpg + k cs, ..) of gate group g, k = block % cpg, dealt to the slots in turn.
// WHOLE (groups shorter than a block's share): every slot owns gps whole groups.  The slots of a block run the
// same number of rows, so that they can share barriers.
struct RowPlan {
    int64_t rpg, cs, cpg, gps, nblocks;
    int whole, W, nw, rpb, threads;
};

RowPlan row_plan(int64_t rows, int64_t C, int64_t gate_groups) {
    RowPlan p = {};
    // 16 lanes a row up to 128 columns, a wave up to 512, then waves (forward + backward, fp32, 16384 x 128: 42 us by
    // 16 lanes, 65 by waves; 8192 x 256: 48.5 by waves, 51.6 by blocks; 8192 x 512: 53.8 / 55.1); past 2048 columns
    // a block has one row and up to 16 waves, with the registers that leaves
    p.W = C <= 128 ? 16 : C <= 512 ? 64 : C <= 2048 ? 0 : C <= 4096 ? -1 : -2;
    p.nw = (int)ceil_div(C, 512);
    p.rpb = p.W > 0 ? 256 / p.W : std::max(1, 4 / p.nw);
    p.threads = p.W > 0 ? 256 : p.rpb * p.nw * 64;
    const int64_t groups = gate_groups > 0 && gate_groups < rows ? gate_groups : 1;
    p.rpg = rows / groups;
    // up to 768 blocks, three on each CU at its 168 registers; each leaves one partial row per sum, read once
    // more.  16384 rows of 2048 bf16 columns, kernel + sums: 109 + 10 us at 512 blocks, 94 + 14 at 768, 110 + 18
    // at 1024 (149 + 19 at four blocks to a CU: the registers spill).  Rows of more than 2048 columns have one block
    // to a CU: 4096 rows of 8192, fp32 188 + 11 us at 256 blocks, 200 + 15 at 512, 213 + 21 at 768 (bf16 223 + 11, 231 +
    // 15, 260 + 22)
    const int64_t chunk = std::max<int64_t>(p.rpb, ceil_div(rows, p.W >= 0 ? 768 : 256));
    p.whole = p.rpg < chunk && groups > 1;
    if (p.whole) {
        p.gps = std::max<int64_t>(1, chunk / p.rpb / p.rpg);
        p.nblocks = ceil_div(ceil_div(groups, p.gps), p.rpb);
        p.cpg = 1;
    } else {
        p.cpg = ceil_div(p.rpg, chunk);
        p.cs = ceil_div(p.rpg, p.cpg);
        p.nblocks = groups * p.cpg;
    }
    return p;
}

// Partial sums per block and column.  A gate shared by a block's rows is taken out of them: SUM_A = sum of du
// yhat (du y without a norm of y), SUM_B = sum of du, du = the gradient behind the gate.  OWN (a gate per row,
// or WHOLE) has the gate inside: SUM_A = sum of dn yhat, SUM_B = sum of dn, dn = du gate.
enum { SUM_A, SUM_B, SUM_PRE_W, SUM_PRE_B, SUMS };

// The backward pass reads y, h, dh and dz once; statistics come from the forward pass.  A 16-bit h has lost what
// xhat needs (the weight gradients would be off by its rounding again), so there x is read in its place and h
// is formed again from x and y.  The same 16384 x 2048 bf16 block: 98 us, 403 MB at 4.1 TB/s, and 9.5 us for the sums.
template <typename TX, typename TY>
struct RowIn {   // a row's eight columns as loaded, one row ahead of their use
    Raw8<TX> dh, h;   // h: x where h is formed again
    Raw8<TY> dz, y;
    float mu1, rs1, mu2, rs2;
    int64_t r;
    int n;
};

template <typename TX, typename TY, int W, bool NORM, bool OWN>
__global__ __launch_bounds__(W >= 0 ? 256 : W == -1 ? 512 : 1024, W >= 0 ? 3 : 1) void residual_norm_bwd_kernel(nbx_residual_norm_args a, RowPlan p,
                                                                                    float keep,
                                                                                    float* __restrict__ part) {
    __shared__ float red[4][16][2];
    __shared__ float comb[W >= 0 ? 2048 : 1];
    int turn = 0;
    const int slot_threads = W > 0 ? W : p.nw * 64;
    // a wave has one row (but for the 16-lane form): the row's addresses and statistics are scalars
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int mine = W == 16 ? (int)threadIdx.x / 16 : W > 0 ? wave : wave / p.nw;
    const int lane = (int)threadIdx.x - mine * slot_threads;
    const int C = (int)a.C, c0 = 8 * lane, cn = std::max(0, std::min(8, C - c0));
    // two sums over a slot's threads at once
    auto slot_sums = [&](float& x, float& y) {
        if constexpr (W > 0) {
            x = lanes_sum<W>(x);
            y = lanes_sum<W>(y);
        } else {
            x = lanes_sum<64>(x);
            y = lanes_sum<64>(y);
            float(*r)[2] = red[turn];
            turn = (turn + 1) & 3;
            if ((threadIdx.x & 63) == 0) {
                r[threadIdx.x >> 6][0] = x;
                r[threadIdx.x >> 6][1] = y;
            }
            __syncthreads();
            x = y = 0.f;
            for (int i = 0; i < p.nw; ++i) {
                x += r[mine * p.nw + i][0];
                y += r[mine * p.nw + i][1];
            }
        }
    };
    Draws d = {{0, 0, 0, 0}, a.threshold, a.group, (a.C + 7) >> 3, keep};
    if (a.threshold) d.key = draw_key(a.rng, a.call);
    const float s = a.scale * keep, invC = 1.0f / (float)C;
    const bool rowgate = OWN && !p.whole, post = NORM && a.post_w, pre = NORM && a.pre_w && a.dz;
    constexpr bool AGAIN = sizeof(TX) == 2;
    // at 16 waves a block (128 registers a thread) no row is fetched ahead and the weights are read per row: 4096 rows
    // of 8192 fp32 columns 188 us, fetched ahead with spills 304.  For 16-bit rows fetching ahead spills less, and is
    // the faster since their norm gradients are formed from x and y (bf16: 189 us against 223 as it is here)
    constexpr bool LEAN = W == -2;
    const bool need_y = post || a.dgate || (AGAIN && pre);
    float acc[SUMS][8] = {}, ag[OWN ? 8 : 1] = {};
    float pw[8], pb[OWN || (AGAIN && NORM) ? 8 : 1] = {}, qw[8], gt[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) gt[i] = 1.f;
    if (post) load8p(a.post_w, a.param_dtype, c0, cn, pw);
    if constexpr (OWN || (AGAIN && NORM))
        if (post && a.post_b) load8p(a.post_b, a.param_dtype, c0, cn, pb);
    if (pre && !LEAN) load8p(a.pre_w, a.param_dtype, c0, cn, qw);
    // the slot's rows: first, past the last, step; all slots of a block run `iters` rows
    int64_t r0, r1, step, iters, left = 0;
    if (p.whole) {
        const int64_t unit = blockIdx.x * (int64_t)p.rpb + mine;
        r0 = std::min(unit * p.gps * p.rpg, a.rows);
        r1 = std::min(r0 + p.gps * p.rpg, a.rows);
        step = 1;
        iters = p.gps * p.rpg;
    } else {
        const int64_t g = blockIdx.x / p.cpg, k0 = blockIdx.x % p.cpg * p.cs;
        r0 = g * p.rpg + k0 + mine;
        r1 = g * p.rpg + std::min(k0 + p.cs, p.rpg);
        step = p.rpb;
        iters = (p.cs + p.rpb - 1) / p.rpb;
        if constexpr (!OWN) {
            if (a.gate) load8p(a.gate, a.param_dtype, g * a.C + c0, cn, gt);
            if (post)   // the norm's weight (and, for h again, its bias) and the gate act on the same values
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (AGAIN && NORM) pb[i] *= gt[i];
                    gt[i] *= pw[i];
                }
        }
    }
    using In = RowIn<TX, TY>;
    auto fetch = [&](int64_t r, In& in) {
        const bool live = r < r1;   // else zeros, its statistics too: nothing of another row reaches the sums
        in.n = live ? cn : 0;
        in.r = live ? r : 0;
        const int64_t row = in.r * a.C;
        fetch8n((const TX*)a.dh + row + (uint32_t)c0, a.dh ? in.n : 0, in.dh);
        if (pre) {
            fetch8n((const TY*)a.dz + row + (uint32_t)c0, in.n, in.dz);
            if constexpr (AGAIN) fetch8n((const TX*)a.x + in.r * a.ldx + (uint32_t)c0, in.n, in.h);
            else fetch8n((const TX*)a.h + row + (uint32_t)c0, in.n, in.h);
            in.mu2 = live ? a.stats[2 * a.rows + in.r] : 0.f;
            in.rs2 = live ? a.stats[3 * a.rows + in.r] : 0.f;
        }
        if (need_y) fetch8n((const TY*)a.y + in.r * a.ldy + (uint32_t)c0, in.n, in.y);
        if (post) {
            in.mu1 = live ? a.stats[in.r] : 0.f;
            in.rs1 = live ? a.stats[a.rows + in.r] : 0.f;
        }
    };
    In in;
    if (!LEAN) fetch(r0, in);
    for (int64_t i = 0; i < iters; ++i) {
        In next;
        if constexpr (LEAN) {
            asm volatile("" ::: "memory");   // what is read per row is not kept in registers over the rows
            fetch(r0 + i * step, in);
            if (pre) load8p(a.pre_w, a.param_dtype, c0, cn, qw);
        } else if (i + 1 < iters) {
            fetch(r0 + (i + 1) * step, next);
        }
        const int n = in.n;
        const int64_t row = in.r * a.C;
        if constexpr (OWN) {
            if (rowgate) load8p(a.gate, a.param_dtype, row + (uint32_t)c0, n, gt);
            else if (left == 0) load8p(a.gate, a.param_dtype, in.r / p.rpg * a.C + c0, n, gt);
        }
        float t[8], v[8], e[8];
        const Keep8 m = row_keep(d, in.r, lane);
        unpack8(in.dh, t);
        if (pre) {
            unpack8(in.h, v);
            if constexpr (AGAIN) {
                float u[8];
                unpack8(in.y, u);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (post) {
                        u[k] = (u[k] - in.mu1) * in.rs1;
                        // gt holds the gate times the weight (OWN: the gate alone)
                        if constexpr (NORM) u[k] = OWN ? (u[k] * pw[k] + pb[k]) * gt[k] : u[k] * gt[k] + pb[k];
                    } else {
                        u[k] *= gt[k];
                    }
                    v[k] = fmaf(s, m.k[k] ? u[k] : 0.f, v[k]);
                }
            }
            unpack8(in.dz, e);
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = (v[k] - in.mu2) * in.rs2;
                acc[SUM_PRE_W][k] += e[k] * v[k];  // past the row e is 0
                acc[SUM_PRE_B][k] += e[k];
                e[k] *= qw[k];   // 0 past the row, as every weight below
                s1 += e[k];
                s2 += e[k] * v[k];
            }
            slot_sums(s1, s2);
            s1 = a.norm ? 0.f : s1 * invC;
            s2 *= invC;
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] += in.rs2 * (e[k] - s1 - v[k] * s2);
        }
        if (a.dx) store8n((TX*)a.dx + row + (uint32_t)c0, n, t);
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = m.k[k] ? s * t[k] : 0.f;
        if (need_y) {
            unpack8(in.y, v);
            if (post)
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = (v[k] - in.mu1) * in.rs1;
        }
        if constexpr (OWN) {
            if (a.dgate) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float u = post ? v[k] * pw[k] + pb[k] : v[k];
                    e[k] = m.k[k] ? t[k] * u : 0.f;   // a dropped place counts 0 whatever it held
                    ag[k] += e[k];
                }
                if (rowgate) store8p(a.dgate, a.param_dtype, row + (uint32_t)c0, n, e);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] *= gt[k];
        }
        if (post || (!OWN && a.dgate))
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                acc[SUM_A][k] = fmaf(t[k], m.k[k] ? v[k] : 0.f, acc[SUM_A][k]);
                acc[SUM_B][k] += t[k];
            }
        if constexpr (!OWN)
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] *= gt[k];
        if (post) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (OWN) t[k] *= pw[k];
                s1 += t[k];
                s2 += t[k] * v[k];
            }
            slot_sums(s1, s2);
            s1 = a.norm ? 0.f : s1 * invC;
            s2 *= invC;
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = in.rs1 * (t[k] - s1 - v[k] * s2);
            if (d.group && !m.k[0])   // the row is dropped, whatever it held: not 0 times an infinity's norm
#pragma unroll
                for (int k = 0; k < 8; ++k) t[k] = 0.f;
        }
        if (a.dy) store8n((TY*)a.dy + row + (uint32_t)c0, n, t);
        if constexpr (OWN) {
            left = left + 1 == p.rpg ? 0 : left + 1;
            if (p.whole && left == 0 && a.dgate) {   // a whole gate group ends: this slot had all of it
                float g[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    g[k] = ag[k];
                    ag[k] = 0.f;
                }
                store8p(a.dgate, a.param_dtype, in.r / p.rpg * a.C + c0, n, g);
            }
        }
        if constexpr (!LEAN) in = next;
    }
    // one partial row per block and sum: part[sum][block][C]
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        const bool want = k == SUM_A ? a.dpost_w || (!OWN && a.dgate) : k == SUM_B ? a.dpost_b || (!OWN && a.dgate && post)
                        : k == SUM_PRE_W ? a.dpre_w != nullptr : a.dpre_b != nullptr;
        if (!want) continue;
        float* to = part + ((int64_t)k * p.nblocks + blockIdx.x) * a.C;
        if (p.rpb == 1) {
            store8n(to + c0, cn, acc[k]);
        } else {
            const int ld = 8 * slot_threads;
            __syncthreads();
            store8(comb + mine * ld + c0, acc[k]);
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += blockDim.x) {
                float t = 0.f;
                for (int q = 0; q < p.rpb; ++q) t += comb[q * ld + c];
                to[c] = t;
            }
        }
    }
}

// Column sums of the partial rows.  The first jobs * ceil(C / 32) blocks: a parameter over all blocks (dpost_*
// with each block's gate row put back), 32 columns x 32 slots, each slot every 32nd row, combined in order.
// Then gate group after group over its cpg blocks: the same, or (cpg <= 16) a thread per column: 64 groups of
// 12 partial rows of 2048 columns, with two parameters: 15.6 us so, 18.3 with slots.
enum { OUT_POST_W, OUT_POST_B, OUT_PRE_W, OUT_PRE_B, OUTS };
struct FinalSums {
    void* out[OUTS];
    void* dgate;
    const void *gate, *post_w, *post_b;   // gate NULL: it is in the sums already
    int dtype, jobs;
    int job[OUTS];
};

__device__ __forceinline__ float load1p(const void* p, int dtype, int64_t at) {
    return dtype == NBX_F32 ? ((const float*)p)[at]
         : dtype == NBX_BF16 ? (float)((const bf16*)p)[at] : (float)((const f16*)p)[at];
}

__global__ __launch_bounds__(1024) void residual_norm_sums_kernel(FinalSums f, int64_t nblocks, int64_t cpg, int64_t C,
                                                                  const float* __restrict__ part) {
    __shared__ float red[2][32][33];
    const int tiles = (int)((C + 31) / 32), job = (int)blockIdx.x / tiles;
    const bool gates = job >= f.jobs, thread_per_column = gates && cpg <= 16;
    const int gtiles = cpg <= 16 ? (int)((C + 1023) / 1024) : tiles, gb = (int)blockIdx.x - f.jobs * tiles;
    const int lane = threadIdx.x & 31, w = thread_per_column ? 0 : threadIdx.x >> 5;
    const int64_t c = thread_per_column ? gb % gtiles * (int64_t)1024 + threadIdx.x
                                        : (gates ? gb % gtiles : (int)blockIdx.x % tiles) * (int64_t)32 + lane;
    const int k = gates ? SUM_A : f.job[job], step = thread_per_column ? 1 : 32;
    const int64_t g = gates ? gb / gtiles : 0;
    const int nb = (int)(gates ? cpg : nblocks);
    const float* p = part + ((int64_t)k * nblocks + g * cpg) * C + c;
    const bool scaled = !gates && f.gate && k <= OUT_POST_B, both = gates && f.post_w;
    float s = 0.f, s2 = 0.f;
    if (c < C) {
        if (scaled) {
            auto with_gate = [&](auto* gate) {
#pragma unroll 8
                for (int b = w; b < nb; b += step) s += p[b * C] * (float)gate[b / (int)cpg * C + c];
            };
            if (f.dtype == NBX_F32) with_gate((const float*)f.gate);
            else if (f.dtype == NBX_BF16) with_gate((const bf16*)f.gate);
            else with_gate((const f16*)f.gate);
        } else if (both) {
#pragma unroll 8
            for (int b = w; b < nb; b += step) {
                s += p[b * C];
                s2 += p[(nblocks + b) * C];
            }
        } else {
#pragma unroll 8
            for (int b = w; b < nb; b += step) s += p[b * C];
        }
    }
    if (!thread_per_column) {
        red[0][w][lane] = s;
        red[1][w][lane] = s2;
        __syncthreads();
        if (w) return;
        s = s2 = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            s += red[0][i][lane];
            s2 += red[1][i][lane];
        }
    }
    if (c >= C) return;
    if (!gates) {
        store1p(f.out[k], f.dtype, c, s);
    } else {
        if (both) s = s * load1p(f.post_w, f.dtype, c) + (f.post_b ? s2 * load1p(f.post_b, f.dtype, c) : 0.f);
        store1p(f.dgate, f.dtype, g * C + c, s);
    }
}

int residual_check(const nbx_residual_norm_args* a, const char* who) {
    NBX_CHECK_ARG(a, "%s: null arguments", who);
    NBX_CHECK_ARG(a->rows >= 0 && a->rows < ((int64_t)1 << 31), "%s: need 0 <= rows < 2^31", who);
    NBX_CHECK_ARG(a->C >= 1 && a->C <= 8192, "%s: need 1 <= C <= 8192", who);
    NBX_CHECK_ARG(dtype_ok(a->x_dtype) && dtype_ok(a->y_dtype) && (a->x_dtype == a->y_dtype || a->x_dtype == NBX_F32),
                  "%s: x_dtype must be y_dtype or fp32", who);
    NBX_CHECK_ARG(a->param_dtype == NBX_F32 || a->param_dtype == a->y_dtype, "%s: param_dtype must be fp32 or y_dtype",
                  who);
    NBX_CHECK_ARG(a->norm == 0 || a->norm == 1, "%s: unknown norm %d", who, a->norm);
    NBX_CHECK_ARG(a->threshold < 65536 && a->group >= 0, "%s: need threshold < 65536, group >= 0", who);
    NBX_CHECK_ARG(!a->threshold || a->rng, "%s: a drop rate needs rng", who);
    NBX_CHECK_ARG(!a->gate || (a->gate_groups >= 1 && (a->rows == 0 || a->rows % a->gate_groups == 0)),
                  "%s: gate_groups must divide rows", who);
    NBX_CHECK_ARG(a->ldy >= a->C && a->ldx >= a->C, "%s: row strides are shorter than the rows", who);
    NBX_CHECK_ARG((!a->post_b || a->post_w) && (!a->pre_b || a->pre_w), "%s: a norm's bias needs its weight", who);
    return NBX_OK;
}

// f(TX{}, TY{}) for the storage types
template <typename F>
int with_types(const nbx_residual_norm_args& a, F&& f) {
    return with_type(a.y_dtype, [&](auto y) {
        using TY = decltype(y);
        if (a.x_dtype == a.y_dtype) return f(TY{}, TY{});
        return f(float{}, TY{});
    });
}

// ======================================================================== residual add, spherical-harmonics norm
// A node's (lmax+1)^2 rows of C channels are cut into chunks of eight channels of one row (the last of a row may
// be shorter), kept in the registers of TPN threads: 64 (four nodes per block) or the block; thread t holds
// chunks t, t + TPN, .. (NJ of them).  The l = 0 row is chunks 0 .. C/8 - 1, all in the first wave, so its
// centring needs no barrier: one block-wide sum per direction is left.  2560 nodes of lmax 6, 128 channels, fp32:
// forward 60 us (257 MB at 4.3 TB/s), backward 67 us (321 MB at 4.8 TB/s) and 4 us for the sums.
constexpr int SH_MAXC = 512;
constexpr int SH_LDS_HEAD = 64 + 2 * 4 * SH_MAXC / 8 / 4;   // floats before the rows in the backward pass's LDS

struct ShPlan {
    int S, cpr, chunks, tpn, nj, npb, threads;   // cpr: chunks per row; npb: nodes in flight per block
};

ShPlan sh_plan(int64_t V, int lmax, int C) {
    ShPlan p = {};
    p.S = (lmax + 1) * (lmax + 1);
    p.cpr = (C + 7) / 8;
    p.chunks = p.S * p.cpr;
    // a wave per node where nodes are many and small; else a block (forward + backward of lmax 2, 64 channels: 320
    // nodes 16.9 us by waves, 14.7 by blocks; 1024: 18.8 / 18.2; 2048: 24.9 / 25.9; 8192: 47 / 68)
    if (p.chunks <= 128 && V >= 2048) {
        p.tpn = 64;
        p.nj = p.chunks <= 64 ? 1 : 2;
        p.npb = 4;
        p.threads = 256;
    } else {
        p.nj = p.chunks <= 1024 ? 1 : p.chunks <= 2048 ? 2 : 4;
        p.tpn = p.threads = (int)ceil_div(ceil_div(p.chunks, p.nj), 64) * 64;
        p.npb = 1;
    }
    return p;
}

// what chunk t + TPN j of a node is
struct ShChunk {
    int at, n, l, c8;   // offset in the node, channels (0: none), degree, channel / 8
    bool first;         // of the l = 0 row
    float bal;
};
__device__ __forceinline__ ShChunk sh_chunk(const ShPlan& p, int q, int C, int lmax) {
    ShChunk k;
    const int i = q / p.cpr;
    k.c8 = q - i * p.cpr;
    k.at = i * C + 8 * k.c8;
    k.n = q < p.chunks ? std::min(8, C - 8 * k.c8) : 0;
    k.l = (i >= 1) + (i >= 4) + (i >= 9) + (i >= 16) + (i >= 25) + (i >= 36);
    k.first = i == 0;
    k.bal = 1.0f / (float)((2 * k.l + 1) * (lmax + 1));
    return k;
}

// sum over a node's threads, in all of them: SUB a wave, else the block (one barrier; `slot` alternates)
template <bool SUB>
__device__ __forceinline__ float node_sum(float x, float (*red)[16], int& slot) {
    return row_sum<SUB ? 64 : 0>(x, red, slot);
}

// the channel draws of a node as bits in LDS: one Philox block per eight channels, shared by its rows
__device__ __forceinline__ void sh_channel_bits(const nbx_sh_residual_norm_args& a, const DrawKey& key, int64_t node,
                                                int t, int cpr, uint8_t* bits) {
    if (t < cpr) bits[t] = (uint8_t)keep_bits(key, (uint64_t)(node * cpr + t), a.channel_threshold);
}

template <typename T, int NJ, bool SUB>
__global__ __launch_bounds__(SUB ? 256 : 1024) void sh_residual_norm_kernel(nbx_sh_residual_norm_args a, ShPlan p,
                                                                            float k1, float k2) {
    __shared__ float red[4][16];
    __shared__ uint8_t bits[SUB ? 4 : 1][SH_MAXC / 8];
    int slot = 0;
    if (a.path_threshold | a.channel_threshold) note_used(a.used, a.rng);
    const int t = SUB ? (int)threadIdx.x & 63 : (int)threadIdx.x, sub = SUB ? (int)threadIdx.x >> 6 : 0;
    const int64_t v = SUB ? blockIdx.x * (int64_t)4 + sub : blockIdx.x;
    const int C = a.C;
    const int64_t base = v * p.S * C;
    const bool live = v < a.V;
    ShChunk q[NJ];
    float h[NJ][8], y[NJ][8];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        q[j] = sh_chunk(p, t + p.tpn * j, C, a.lmax);
        if (!live) q[j].n = 0;
        load8n((const T*)a.x + base + q[j].at, q[j].n, h[j]);
        load8n((const T*)a.y + base + q[j].at, q[j].n, y[j]);
    }
    if (a.channel_threshold) {
        if (live) sh_channel_bits(a, draw_key(a.rng, a.call + 1), v, t, p.cpr, bits[sub]);
        __syncthreads();
    }
    if (!live) return;   // SUB: whole waves, no barrier below
    float k = a.channel_threshold ? k2 : 1.f;
    uint32_t path = 0xFFu;
    if (a.path_threshold) {
        k *= k1;
        path = keep_one(draw_key(a.rng, a.call), (uint64_t)(v / a.path_group), a.path_threshold) ? 0xFFu : 0u;
    }
    float s0 = 0.f, qs = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const uint32_t m = a.channel_threshold ? path & bits[sub][q[j].c8] : path;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[j][e] += (m >> e & 1) ? k * y[j][e] : 0.f;   // past the row: 0
            s += h[j][e] * h[j][e];
            if (j == 0 && q[0].first) s0 += h[0][e];
        }
        if (!q[j].first) qs += q[j].bal * s;
        store8n((T*)a.h + base + q[j].at, q[j].n, h[j]);
    }
    float m0 = 0.f;
    if (t < 64) {   // the first wave holds the l = 0 row
        m0 = lanes_sum<64>(s0) / (float)C;
        if (q[0].first) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[0][e] -= m0;
                if (e < q[0].n) s += h[0][e] * h[0][e];
            }
            qs += q[0].bal * s;
        }
    }
    const float rs = 1.0f / sqrtf(node_sum<SUB>(qs, red, slot) / (float)C + a.eps);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        float w[8];
        load8p(a.weight, a.param_dtype, q[j].l * C + 8 * q[j].c8, q[j].n, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[j][e] = h[j][e] * rs * w[e];
        if (j == 0 && q[0].first) {
            load8p(a.bias, a.param_dtype, 8 * q[0].c8, q[0].n, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[0][e] += w[e];
        }
        store8n((T*)a.z + base + q[j].at, q[j].n, h[j]);
    }
    if (a.stats && t == 0) {
        a.stats[v] = m0;
        a.stats[a.V + v] = rs;
    }
}

// Backward over nodes unit, unit + nunits, ..: each thread keeps its chunks' weights, and the column sums of
// dz hc rs per row and of dz's l = 0 row, in registers over the nodes.  At the end the rows of a degree are
// summed in LDS: part[unit][(lmax + 2) C] = (dweight | dbias) of the unit's nodes.
template <typename T, int NJ, bool SUB>
__global__ __launch_bounds__(SUB ? 256 : 1024) void sh_residual_norm_bwd_kernel(nbx_sh_residual_norm_args a, ShPlan p,
                                                                                float k1, float k2, int64_t nunits,
                                                                                float* __restrict__ part) {
    // all of it dynamic, so that the kernel's limit can be raised to the whole 160 KB
    extern __shared__ float sh_lds[];
    float (*red)[16] = reinterpret_cast<float (*)[16]>(sh_lds);                        // [4][16]
    auto bits = reinterpret_cast<uint8_t (*)[SUB ? 4 : 1][SH_MAXC / 8]>(sh_lds + 64);   // [2]
    float* rows = sh_lds + SH_LDS_HEAD;                                                // [npb][chunks 8]
    int slot = 0, flip = 0;
    const int t = SUB ? (int)threadIdx.x & 63 : (int)threadIdx.x, sub = SUB ? (int)threadIdx.x >> 6 : 0;
    const int64_t unit = SUB ? blockIdx.x * (int64_t)4 + sub : blockIdx.x;
    const int C = a.C;
    constexpr bool AGAIN = sizeof(T) == 2;   // a 16-bit h has lost what the norm's gradient needs: x + k y again
    const float k = (a.path_threshold ? k1 : 1.f) * (a.channel_threshold ? k2 : 1.f);
    DrawKey key = {0, 0, 0, 0};
    if (a.path_threshold | a.channel_threshold) key = draw_key(a.rng, a.call);
    ShChunk q[NJ];
    float w[NJ][8], aw[NJ][8] = {}, ab[8] = {};
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        q[j] = sh_chunk(p, t + p.tpn * j, C, a.lmax);
        load8p(a.weight, a.param_dtype, q[j].l * C + 8 * q[j].c8, q[j].n, w[j]);
    }
    const int64_t iters = (a.V + nunits - 1) / nunits;
    for (int64_t it = 0; it < iters; ++it) {
        const int64_t v = it * nunits + unit;
        const bool live = v < a.V;
        if (a.channel_threshold) {   // two copies: the next node's bits are written before this one's last read
            DrawKey ck = key;
            ck.call = a.call + 1;
            if (live) sh_channel_bits(a, ck, v, t, p.cpr, bits[flip][sub]);
            __syncthreads();
        }
        const uint8_t* bt = bits[flip][sub];
        flip ^= 1;
        if (!live) {
            if (SUB) continue;
            break;   // the whole block
        }
        const int64_t base = v * p.S * C;
        const float m0 = a.stats[v], rs = a.stats[a.V + v];
        float g[NJ][8], hc[NJ][8], dh[NJ][8];
        float dot = 0.f, sg = 0.f;
        uint32_t path = 0xFFu;
        if (a.path_threshold)
            path = keep_one(key, (uint64_t)(v / a.path_group), a.path_threshold) ? 0xFFu : 0u;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = q[j].n;
            load8n((const T*)a.dz + base + q[j].at, a.dz ? n : 0, g[j]);
            load8n((const T*)(AGAIN ? a.x : a.h) + base + q[j].at, a.dz ? n : 0, hc[j]);
            load8n((const T*)a.dh + base + q[j].at, a.dh ? n : 0, dh[j]);
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (AGAIN) {
                const uint32_t m = a.channel_threshold ? path & bt[q[j].c8] : path;
                float y[8];
                load8n((const T*)a.y + base + q[j].at, a.dz ? q[j].n : 0, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) hc[j][e] += (m >> e & 1) ? k * y[e] : 0.f;
            }
            if (j == 0 && q[0].first) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (e < q[0].n) hc[0][e] -= m0;
                    ab[e] += g[0][e];
                    sg += g[0][e] * w[0][e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                hc[j][e] *= rs;
                aw[j][e] += g[j][e] * hc[j][e];
                g[j][e] *= w[j][e];
                dot += g[j][e] * hc[j][e];
            }
        }
        dot = node_sum<SUB>(dot, red, slot) / (float)C;
        // the centred row sums to 0, so only g is left of the l = 0 row's mean
        const float dm = t < 64 ? lanes_sum<64>(sg) / (float)C : 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const uint32_t m = a.channel_threshold ? path & bt[q[j].c8] : path;
            const float cb = dot * q[j].bal, d0 = q[j].first ? dm : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = dh[j][e] + rs * (g[j][e] - cb * hc[j][e] - d0);
                g[j][e] = d;
                hc[j][e] = (m >> e & 1) ? k * d : 0.f;
            }
            if (a.dx) store8n((T*)a.dx + base + q[j].at, q[j].n, g[j]);
            if (a.dy) store8n((T*)a.dy + base + q[j].at, q[j].n, hc[j]);
        }
    }
    if (!part) return;
    const int row = 8 * p.cpr;
    float* mine = rows + sub * 8 * p.chunks;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
        if (q[j].n) store8(mine + 8 * (t + p.tpn * j), aw[j]);
    float* to = part + unit * (int64_t)(a.lmax + 2) * C;
    if (q[0].first && q[0].n) store8n(to + (a.lmax + 1) * C + 8 * q[0].c8, q[0].n, ab);
    __syncthreads();
    for (int o = t; o < (a.lmax + 1) * C; o += p.tpn) {
        const int l = o / C, c = o - l * C;
        float s = 0.f;
        for (int i = l * l; i < (l + 1) * (l + 1); ++i) s += mine[i * row + c];
        to[o] = s;
    }
}

// dweight [lmax+1][C] | dbias [C] from the units' partial rows: 32 columns x 32 slots in a fixed order
__global__ __launch_bounds__(1024) void sh_residual_sums_kernel(nbx_sh_residual_norm_args a, int64_t nunits,
                                                                const float* __restrict__ part) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t ld = (int64_t)(a.lmax + 2) * a.C;
    const int64_t c = blockIdx.x * (int64_t)32 + lane;
    float s = 0.f;
    if (c < ld)
#pragma unroll 8
        for (int64_t u = w; u < nunits; u += 32) s += part[u * ld + c];
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < ld) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += red[i][lane];
        const int64_t nw = ld - a.C;
        if (c < nw) {
            if (a.dweight) store1p(a.dweight, a.param_dtype, c, t);
        } else if (a.dbias) {
            store1p(a.dbias, a.param_dtype, c - nw, t);
        }
    }
}

// the units (nodes in flight) of the backward pass: its partial rows are read and written once more
int64_t sh_units(const ShPlan& p, int64_t V) {
    const int64_t most = 512 * (int64_t)p.npb;
    return ceil_div(std::min(most, V), p.npb) * p.npb;
}

size_t sh_workspace(const ShPlan& p, int64_t V, int lmax, int C) {
    return (size_t)sh_units(p, V) * (lmax + 2) * C * sizeof(float);
}

int sh_check(const nbx_sh_residual_norm_args* a, const char* who) {
    NBX_CHECK_ARG(a, "%s: null arguments", who);
    NBX_CHECK_ARG(a->V >= 0 && a->V < ((int64_t)1 << 31) && a->lmax >= 0 && a->lmax <= 6 && a->C >= 1 && a->C <= SH_MAXC,
                  "%s: need 0 <= V < 2^31, 0 <= lmax <= 6, 1 <= C <= %d", who, SH_MAXC);
    NBX_CHECK_ARG(dtype_ok(a->dtype) && (a->param_dtype == NBX_F32 || a->param_dtype == a->dtype),
                  "%s: param_dtype must be fp32 or dtype", who);
    NBX_CHECK_ARG(a->path_threshold < 65536 && a->channel_threshold < 65536 && a->path_group >= 1,
                  "%s: need thresholds < 65536, path_group >= 1", who);
    NBX_CHECK_ARG(!(a->path_threshold | a->channel_threshold) || a->rng, "%s: a drop rate needs rng", who);
    NBX_CHECK_ARG(a->V == 0 || a->weight, "%s: null weight", who);
    return NBX_OK;
}

template <bool BWD, typename T>
int sh_launch(const nbx_sh_residual_norm_args& a, const ShPlan& p, int64_t units, float* part, hipStream_t st) {
    const float k1 = keep_scale(a.path_threshold), k2 = keep_scale(a.channel_threshold);
    const unsigned blocks = (unsigned)ceil_div(BWD ? units : a.V, p.npb);
    auto go = [&](auto fwd, auto bwd) {
        if constexpr (BWD) {
            // up to 98 KB of LDS (lmax 6, 512 channels)
            const size_t lds = (SH_LDS_HEAD + (part ? (size_t)p.npb * p.chunks * 8 : 0)) * sizeof(float);
            if (lds > 60 * 1024) NBX_LDS_160K(bwd);
            hipLaunchKernelGGL(bwd, dim3(blocks), dim3(p.threads), lds, st, a, p, k1, k2, units, part);
        } else {
            hipLaunchKernelGGL(fwd, dim3(blocks), dim3(p.threads), 0, st, a, p, k1, k2);
        }
        return NBX_OK;
    };
    if (p.npb == 4) {
        if (p.nj == 1) return go(sh_residual_norm_kernel<T, 1, true>, sh_residual_norm_bwd_kernel<T, 1, true>);
        return go(sh_residual_norm_kernel<T, 2, true>, sh_residual_norm_bwd_kernel<T, 2, true>);
    }
    if (p.nj == 1) return go(sh_residual_norm_kernel<T, 1, false>, sh_residual_norm_bwd_kernel<T, 1, false>);
    if (p.nj == 2) return go(sh_residual_norm_kernel<T, 2, false>, sh_residual_norm_bwd_kernel<T, 2, false>);
    return go(sh_residual_norm_kernel<T, 4, false>, sh_residual_norm_bwd_kernel<T, 4, false>);
}

}  // namespace

// ======================================================================== C ABI (include/nbx.h)
extern "C" int nbx_dropout(int32_t dtype, int32_t per, int64_t n, int64_t S, int64_t C, int64_t group,
                           uint32_t threshold, const int64_t* rng, uint32_t call, int64_t* used, const void* X, void* Y,
                           void* stream) {
    NBX_CHECK_ARG(dtype_ok(dtype), "nbx_dropout: unknown dtype %d", dtype);
    NBX_CHECK_ARG(per >= NBX_DROP_ELEMENT && per <= NBX_DROP_CHANNEL, "nbx_dropout: unknown mode %d", per);
    NBX_CHECK_ARG(n >= 0 && S >= 0 && C >= 0 && group >= 1, "nbx_dropout: bad sizes");
    NBX_CHECK_ARG(threshold < 65536, "nbx_dropout: need threshold < 65536");
    if (n == 0 || S == 0 || C == 0) return NBX_OK;
    const int64_t limit = (int64_t)1 << 40;
    NBX_CHECK_ARG(n <= limit && S <= limit / n && C <= limit / (n * S), "nbx_dropout: need n S C <= 2^40");
    NBX_CHECK_ARG(X && Y && rng, "nbx_dropout: null operand");
    hipStream_t st = (hipStream_t)stream;
    const float scale = keep_scale(threshold);
    const int64_t total = n * S * C, RS = S * C;
    return with_type(dtype, [&](auto tag) -> int {
        using T = decltype(tag);
        if (per == NBX_DROP_ELEMENT) {
            const int64_t blocks = ceil_div(total, 2048);
            NBX_CHECK_ARG(grid_ok(blocks, 256), "nbx_dropout: too many elements");
            hipLaunchKernelGGL(dropout_flat_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, total, threshold, scale,
                               rng, call, used, (const T*)X, (T*)Y);
        } else {
            const bool channel = per == NBX_DROP_CHANNEL;
            const int64_t chunks = ceil_div(RS, 8);
            int rpb = chunks <= 128 ? (int)(256 / chunks) : 1;
            const int64_t segs = rpb > 1 ? 1 : ceil_div(chunks, 256), blocks = ceil_div(n, rpb) * segs;
            NBX_CHECK_ARG(grid_ok(blocks, 256), "nbx_dropout: too many elements");
            const int cpr = rpb > 1 ? (int)chunks : 256;
            if (channel)
                hipLaunchKernelGGL((dropout_rows_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, n, RS, C, group, cpr, rpb, segs, threshold, scale, rng, call,
                                   used, (const T*)X, (T*)Y);
            else
                hipLaunchKernelGGL((dropout_rows_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, n, RS, C,
                                   group, cpr, rpb, segs, threshold, scale, rng, call, used, (const T*)X, (T*)Y);
        }
        NBX_LAUNCH_CHECK("dropout");
        return NBX_OK;
    });
}

extern "C" int nbx_residual_norm(const nbx_residual_norm_args* a, void* stream) {
    if (int rc = residual_check(a, "nbx_residual_norm")) return rc;
    if (a->rows == 0) return NBX_OK;
    NBX_CHECK_ARG(a->x && a->y && a->h && (!a->pre_w || a->z), "nbx_residual_norm: null operand");
    const int W = a->C <= 128 ? 16 : a->C <= 512 ? 64 : 0, threads = W ? 256 : (int)ceil_div(a->C, 512) * 64;
    const int64_t blocks = ceil_div(a->rows, W ? 256 / W : 1);
    NBX_CHECK_ARG(grid_ok(blocks, threads), "nbx_residual_norm: too many rows");
    const float keep = keep_scale(a->threshold);
    return with_types(*a, [&](auto x, auto y) -> int {
        using TX = decltype(x);
        using TY = decltype(y);
        auto k = W == 16 ? residual_norm_kernel<TX, TY, 16> : W == 64 ? residual_norm_kernel<TX, TY, 64>
                                                                      : residual_norm_kernel<TX, TY, 0>;
        hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(threads), 0, (hipStream_t)stream, *a, keep);
        NBX_LAUNCH_CHECK("residual_norm");
        return NBX_OK;
    });
}

extern "C" int nbx_residual_norm_backward_workspace_bytes(const nbx_residual_norm_args* a, size_t* bytes) {
    if (int rc = residual_check(a, "nbx_residual_norm_backward_workspace_bytes")) return rc;
    NBX_CHECK_ARG(bytes, "nbx_residual_norm_backward_workspace_bytes: null result");
    *bytes = a->rows ? (size_t)SUMS * row_plan(a->rows, a->C, a->gate ? a->gate_groups : 0).nblocks * a->C * sizeof(float)
                     : 0;
    return NBX_OK;
}

extern "C" int nbx_residual_norm_backward(const nbx_residual_norm_args* a, void* stream) {
    if (int rc = residual_check(a, "nbx_residual_norm_backward")) return rc;
    NBX_CHECK_ARG(a->rows >= 1, "nbx_residual_norm_backward: need a row");
    NBX_CHECK_ARG((!a->post_w && !a->dgate) || a->y, "nbx_residual_norm_backward: null y");
    const bool again = a->x_dtype != NBX_F32;   // h is formed again from x and y
    NBX_CHECK_ARG(!a->pre_w || !a->dz || (again ? a->x && a->y : a->h != nullptr), "nbx_residual_norm_backward: null h");
    NBX_CHECK_ARG((!a->pre_w && !a->post_w) || a->stats, "nbx_residual_norm_backward: null stats");
    NBX_CHECK_ARG((!a->dgate || a->gate) && ((!a->dpost_w && !a->dpost_b) || a->post_w) &&
                      ((!a->dpre_w && !a->dpre_b) || a->pre_w),
                  "nbx_residual_norm_backward: a gradient of a parameter that is not there");
    const int64_t rows = a->rows, C = a->C;
    const RowPlan p = row_plan(rows, C, a->gate ? a->gate_groups : 0);
    const size_t need = (size_t)SUMS * p.nblocks * C * sizeof(float);
    if (!(a->workspace && a->workspace_bytes >= need)) {
        set_error("nbx_residual_norm_backward: workspace too small");
        return NBX_E_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    const float keep = keep_scale(a->threshold);
    float* part = (float*)a->workspace;
    const bool own = a->gate && (p.whole || (a->gate_groups == rows && rows > 1));
    if (int rc = with_types(*a, [&](auto x, auto y) -> int {
            using TX = decltype(x);
            using TY = decltype(y);
            const bool norm = a->post_w || a->pre_w;
            auto pick = [&](auto w) {
                constexpr int W = decltype(w)::value;
                return norm ? (own ? residual_norm_bwd_kernel<TX, TY, W, true, true> : residual_norm_bwd_kernel<TX, TY, W, true, false>)
                            : (own ? residual_norm_bwd_kernel<TX, TY, W, false, true> : residual_norm_bwd_kernel<TX, TY, W, false, false>);
            };
            auto k = p.W == 16 ? pick(std::integral_constant<int, 16>{}) : p.W == 64 ? pick(std::integral_constant<int, 64>{})
                   : p.W == 0 ? pick(std::integral_constant<int, 0>{}) : p.W == -1 ? pick(std::integral_constant<int, -1>{})
                                                                                                : pick(std::integral_constant<int, -2>{});
            hipLaunchKernelGGL(k, dim3((unsigned)p.nblocks), dim3(p.threads), 0, st, *a, p, keep, part);
            NBX_LAUNCH_CHECK("residual_norm_bwd");
            return NBX_OK;
        }))
        return rc;
    FinalSums f = {{a->dpost_w, a->dpost_b, a->dpre_w, a->dpre_b}, a->dgate, own ? nullptr : a->gate, a->post_w, a->post_b,
                   a->param_dtype, 0, {}};
    for (int k = 0; k < OUTS; ++k)
        if (f.out[k]) f.job[f.jobs++] = k;
    const int64_t blocks = f.jobs * ceil_div(C, 32) +
                           (a->dgate && !own ? a->gate_groups * ceil_div(C, p.cpg <= 16 ? 1024 : 32) : 0);
    if (blocks) {
        hipLaunchKernelGGL(residual_norm_sums_kernel, dim3((unsigned)blocks), dim3(1024), 0, st, f, p.nblocks, p.cpg, C,
                           part);
        NBX_LAUNCH_CHECK("residual_norm_sums");
    }
    return NBX_OK;
}

extern "C" int nbx_sh_residual_norm(const nbx_sh_residual_norm_args* a, void* stream) {
    if (int rc = sh_check(a, "nbx_sh_residual_norm")) return rc;
    if (a->V == 0) return NBX_OK;
    NBX_CHECK_ARG(a->x && a->y && a->bias && a->h && a->z, "nbx_sh_residual_norm: null operand");
    const ShPlan p = sh_plan(a->V, a->lmax, a->C);
    NBX_CHECK_ARG(grid_ok(ceil_div(a->V, p.npb), p.threads), "nbx_sh_residual_norm: too many nodes");
    if (int rc = with_type(a->dtype, [&](auto t) { return sh_launch<false, decltype(t)>(*a, p, 0, nullptr, (hipStream_t)stream); }))
        return rc;
    NBX_LAUNCH_CHECK("sh_residual_norm");
    return NBX_OK;
}

extern "C" int nbx_sh_residual_norm_backward_workspace_bytes(const nbx_sh_residual_norm_args* a, size_t* bytes) {
    if (int rc = sh_check(a, "nbx_sh_residual_norm_backward_workspace_bytes")) return rc;
    NBX_CHECK_ARG(bytes, "nbx_sh_residual_norm_backward_workspace_bytes: null result");
    const ShPlan p = sh_plan(a->V, a->lmax, a->C);
    *bytes = a->V ? sh_workspace(p, a->V, a->lmax, a->C) : 0;
    return NBX_OK;
}

extern "C" int nbx_sh_residual_norm_backward(const nbx_sh_residual_norm_args* a, void* stream) {
    if (int rc = sh_check(a, "nbx_sh_residual_norm_backward")) return rc;
    NBX_CHECK_ARG(a->V >= 1, "nbx_sh_residual_norm_backward: need a node");
    NBX_CHECK_ARG(a->stats && (!a->dz || (a->dtype == NBX_F32 ? a->h != nullptr : a->x && a->y)),
                  "nbx_sh_residual_norm_backward: null operand");
    const ShPlan p = sh_plan(a->V, a->lmax, a->C);
    const int64_t units = sh_units(p, a->V);
    const bool sums = a->dweight || a->dbias;
    if (sums && !(a->workspace && a->workspace_bytes >= sh_workspace(p, a->V, a->lmax, a->C))) {
        set_error("nbx_sh_residual_norm_backward: workspace too small");
        return NBX_E_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    float* part = sums ? (float*)a->workspace : nullptr;
    if (int rc = with_type(a->dtype, [&](auto t) { return sh_launch<true, decltype(t)>(*a, p, units, part, st); })) return rc;
    NBX_LAUNCH_CHECK("sh_residual_norm_bwd");
    if (sums) {
        hipLaunchKernelGGL(sh_residual_sums_kernel, dim3((unsigned)ceil_div((a->lmax + 2) * a->C, 32)), dim3(1024), 0, st,
                           *a, units, part);
        NBX_LAUNCH_CHECK("sh_residual_sums");
    }
    return NBX_OK;
}
