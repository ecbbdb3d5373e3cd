// Attention of a step of drafted tokens (include/det_b200.h, det_ftree_op): one pass over the keys with the running maximum and sum of
// the softmax, in 32-bit.  ftree.cuh says how the work is dealt out.
//
//   k_ftree_few    bfloat16, few rows or short caches: ftree_few.cu.
//   k_ftree_tc     bfloat16: ftree_tc.cu.
//   k_ftree_simt   fp32: products on the CUDA cores, 256 threads over a tile of query rows x 32 keys.
//   k_ftree_merge  adds the pieces of the segments that several CTAs shared.
#include "ftree.cuh"
#include <algorithm>
#include <cmath>

namespace detb {

constexpr int TS_KEYS = 32, TS_NJ = TS_KEYS / 16, TS_THREADS = 256;
constexpr int TS_LDS = TS_KEYS + 8, TS_FEW = 4 * 16 * TS_LDS + 16;      // blocks of 16 rows: partial scores, factors

// Of a CTA: query rows, two stages of keys and values, weights (208,896 bytes at most: 64 rows, heads of 256).
static size_t simt_smem(int block, int kd, int vd) {
    return ((size_t)block * (kd + 4) + (size_t)2 * TS_KEYS * (kd + vd + 8) + (size_t)block * (TS_KEYS + 4) + (block == 16 ? TS_FEW : 0)) * sizeof(float);
}
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float dot4(float4 a, float4 b, float s) {
    return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s))));
}
// maximum and sum over the 16 lanes that share a row
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, off));
    return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) v += __shfl_xor_sync(FULL, v, off);
    return v;
}
__device__ __forceinline__ void copy16(float* dst, const float* src, int bytes) {      // what is missing of 16 bytes becomes zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes) : "memory");
}
// The 32 rows of a tile, n floats (a multiple of 4) each, `ld` apart, into rows of n + 4; rows past `have` become zeros.  LANES threads take
// the 16-byte pieces of a row, so an address is one addition.
template <int LANES>
__device__ __forceinline__ void copy_tile(float* dst, const float* src, size_t ld, int n, int have) {
    constexpr int STEP = TS_THREADS / LANES;
    const int c = (threadIdx.x % LANES) * 4, r0 = threadIdx.x / LANES;
    if (c >= n) return;
    const float* first = src + c;
    src += r0 * ld + c;
    dst += r0 * (n + 4) + c;
    const size_t step = STEP * ld;
    const int to = STEP * (n + 4);
    if (have >= TS_KEYS) {
#pragma unroll
        for (int i = 0; i < TS_KEYS / STEP; i++, src += step, dst += to) copy16(dst, src, 16);
    } else {
        for (int r = r0; r < TS_KEYS; r += STEP, src += step, dst += to) copy16(dst, r < have ? src : first, r < have ? 16 : 0);
    }
}
__device__ __forceinline__ void copy_tile(float* dst, const float* src, size_t ld, int n, int have) {
    if (n <= 32) copy_tile<8>(dst, src, ld, n, have);
    else if (n <= 64) copy_tile<16>(dst, src, ld, n, have);
    else if (n <= 128) copy_tile<32>(dst, src, ld, n, have);
    else copy_tile<64>(dst, src, ld, n, have);
}

// Thread (ty, tx) of 16 x 16 has rows ty + 16 i, keys tx + 16 j and value columns 4 tx + 64 j.  Two stages: the next tile's copies run
// beside the products of this one; two CTAs on an SM cover one another's latencies.  Bound by the fp32 multiply-adds and their operands
// from shared memory where keys are many (a key costs all rows of the block, 16 TR, whatever is in them: 16 nodes of 4 sequences behind 4096
// keys, 40 / 8 heads of 128, 255 us), by start, deal and second launch where they are few (6 / 2 heads of 40 and 24, five trees of 13
// nodes behind 2000 keys: 22.7 us; when it was 23.8, tiles of 64 keys and one CTA on an SM took 27.7).
template <int TR, int VJ, bool FEW>
__global__ void __launch_bounds__(TS_THREADS, VJ < 4 ? 2 : 1) k_ftree_simt(const TreeArgs a) {
    extern __shared__ __align__(16) float tsm[];
    __shared__ TreeShare share;
    __shared__ int odd;                          // a staged value that not every row sees was not finite
    constexpr int RB = 16 * TR, LDP = TS_KEYS + 4;
    const int ldk = a.kd + 4, ldv = a.vd + 4, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    float* Q = tsm;                              // [RB][ldk]
    float* P = Q + RB * ldk;                     // [RB][LDP]
    float* KV = P + RB * LDP;                    // [stage] K [32][ldk] | V [32][ldv]
    const int stage_floats = TS_KEYS * (ldk + ldv);
    // lanes that a row's values need; with fewer than 16 the others take other keys (a run of 4 after the other goes round)
    const int lv = FEW || VJ > 1 || a.vd > 32 ? 16 : a.vd > 16 ? 8 : 4, vx = tx & (lv - 1), kstep = 64 / lv;
    // FEW (16 rows): every warp would read all keys for two rows of its own, so here a warp has all rows, 16 keys and a quarter of the elements
    // of the scores, and four keys of the values; what the warps have is added up per tile and per stretch
    constexpr int NQ = VJ == 4 ? 2 : 1, KPL = VJ == 1 ? 2 : 4;           // a lane's columns in fours, its keys
    const int warp = tid >> 5, lane = tid & 31, fc = (VJ == 1 ? lane & 15 : lane) * 4, fk = warp * 4 + (VJ == 1 ? (lane >> 4) * 2 : 0);
    float* S4 = KV + 2 * stage_floats;      // [quarter][16][TS_LDS]
    float* Fs = S4 + 4 * 16 * TS_LDS;            // a row's factor
    pdl_wait();
    pdl_trigger();                               // behind the wait: what k_ftree_merge reads ahead of its own is then there
    if (tid < 32) {
        const TreeShare w = tree_start(a, blockIdx.x, tid);
        if (tid == 0) share = w;
    }
    __syncthreads();
    TreeWalk walk{share, false};
    TreeItem it;
    while (tree_next(a, walk, it)) {
        const TreeSeg& s = it.s;
        const float* cache = static_cast<const float*>(a.seq.table[s.b].cache);
        const float* q = static_cast<const float*>(a.q) + (size_t)s.first * a.ldq + (size_t)it.g * a.per_kv * a.kd;
        auto fetch = [&](int t, int stage) {
            if (t < it.tile + it.n) {
                const int k0 = t * TS_KEYS, have = s.len + s.n - k0;
                const float* rows = cache + (size_t)k0 * a.ld;
                copy_tile(KV + stage * stage_floats, rows + it.g * a.kd, a.ld, a.kd, have);
                copy_tile(KV + stage * stage_floats + TS_KEYS * ldk, rows + a.kv_heads * a.kd + it.g * a.vd, a.ld, a.vd, have);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();
        if (tid == 0) odd = 0;
        fetch(it.tile, 0);
        for (int i = tid; i < RB * (a.kd / 4); i += TS_THREADS) {
            const int r = i / (a.kd / 4), e = (i - r * (a.kd / 4)) * 4, row = s.r0 + r, node = (int)(row * a.per_magic >> 32);
            float4 v = make_float4(0, 0, 0, 0);
            if (r < s.rows) v = load4(q + (size_t)node * a.ldq + (row - node * a.per_kv) * a.kd + e);
            put4(Q + r * ldk + e, v);
        }
        float m[TR], l[TR];
        float4 o[TR][VJ];
#pragma unroll
        for (int i = 0; i < TR; i++) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < VJ; j++) o[i][j] = make_float4(0, 0, 0, 0);
        }
        float4 acc[FEW ? 16 : 1][NQ];
#pragma unroll
        for (int r = 0; r < (FEW ? 16 : 1); r++)
#pragma unroll
            for (int n = 0; n < NQ; n++) acc[r][n] = make_float4(0, 0, 0, 0);
        for (int t = it.tile, stage = 0; t < it.tile + it.n; t++, stage ^= 1) {
            const int k0 = t * TS_KEYS;
            const bool tree = k0 + TS_KEYS > s.edge;
            float* K = KV + stage * stage_floats;
            float* V = K + TS_KEYS * ldk;
            fetch(t + 1, stage ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();
            if (tree) {                          // a weight of zero does not undo a value that is not finite
                for (int i = tid; i < TS_KEYS * a.vd; i += TS_THREADS) {
                    float* p = V + i / a.vd * ldv + i % a.vd;
                    if (!isfinite(*p)) *p = 0.0f, odd = 1;
                }
            }
            float sc[TR][TS_NJ];
#pragma unroll
            for (int i = 0; i < TR; i++)
#pragma unroll
                for (int j = 0; j < TS_NJ; j++) sc[i][j] = 0.0f;
            if constexpr (FEW) {
                const int rg = lane >> 3, kg = (warp & 1) * 16 + (lane & 7), quarter = warp >> 1;
                float part[4][2] = {};
#pragma unroll 1
                for (int e = quarter * 4; e < a.kd; e += 16) {
                    const float4 k0v = load4(K + kg * ldk + e), k1v = load4(K + (kg + 8) * ldk + e);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 qv = load4(Q + (rg + 4 * i) * ldk + e);
                        part[i][0] = dot4(qv, k0v, part[i][0]);
                        part[i][1] = dot4(qv, k1v, part[i][1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) S4[(quarter * 16 + rg + 4 * i) * TS_LDS + kg + 8 * j] = part[i][j];
                __syncthreads();
#pragma unroll
                for (int j = 0; j < TS_NJ; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) sc[0][j] += S4[(c * 16 + ty) * TS_LDS + tx + 16 * j];
            } else {
#pragma unroll 2
                for (int e = 0; e < a.kd; e += 4) {
                    float4 kv[TS_NJ];
#pragma unroll
                    for (int j = 0; j < TS_NJ; j++) kv[j] = load4(K + (tx + 16 * j) * ldk + e);
#pragma unroll
                    for (int i = 0; i < TR; i++) {
                        const float4 qv = load4(Q + (ty + 16 * i) * ldk + e);
#pragma unroll
                        for (int j = 0; j < TS_NJ; j++) sc[i][j] = dot4(qv, kv[j], sc[i][j]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < TR; i++) {
                const int r = ty + 16 * i;
                unsigned seen[TS_KEYS / 32];
#pragma unroll
                for (int j = 0; j < TS_KEYS / 32; j++) seen[j] = FULL;
                if (tree) {
                    const int row = s.r0 + min(r, s.rows - 1);
                    tree_seen<TS_KEYS / 32>(a, s, (int)(row * a.per_magic >> 32), k0, seen);
                }
                float mx = m[i];
#pragma unroll
                for (int j = 0; j < TS_NJ; j++) {
                    sc[i][j] = (seen[j >> 1] >> (tx + 16 * (j & 1))) & 1u ? sc[i][j] * a.scale2 : -INFINITY;
                    mx = fmaxf(mx, sc[i][j]);
                }
                mx = row_max(mx);
                const float base = mx == -INFINITY ? 0.0f : mx, f = exp2f(m[i] - base);
                m[i] = mx;
                l[i] *= f;
                if constexpr (FEW) {
                    if (tx == 0) Fs[ty] = f;
                } else {
#pragma unroll
                    for (int j = 0; j < VJ; j++) o[i][j] = scaled4(o[i][j], f);
                }
#pragma unroll
                for (int j = 0; j < TS_NJ; j++) {
                    const float p = exp2f(sc[i][j] - base);
                    l[i] += p;
                    P[r * LDP + tx + 16 * j] = p;
                }
            }
            __syncthreads();
            if constexpr (FEW) {
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    if (fc + 128 * n >= a.vd) continue;
                    float4 v[KPL];
#pragma unroll
                    for (int k = 0; k < KPL; k++) v[k] = load4(V + (fk + k) * ldv + fc + 128 * n);
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        acc[r][n] = scaled4(acc[r][n], Fs[r]);
                        const float* p = P + r * LDP + fk;
                        if (KPL == 4) {
                            const float4 w = load4(p);
                            add4(acc[r][n], w.x, v[0]);
                            add4(acc[r][n], w.y, v[1]);
                            add4(acc[r][n], w.z, v[KPL - 2]);
                            add4(acc[r][n], w.w, v[KPL - 1]);
                        } else {
                            const float2 w = *reinterpret_cast<const float2*>(p);
                            add4(acc[r][n], w.x, v[0]);
                            add4(acc[r][n], w.y, v[1]);
                        }
                    }
                }
            } else {
                for (int k = tx / lv * 4; k < TS_KEYS; k += kstep) {
                    float4 p[TR];
#pragma unroll
                    for (int i = 0; i < TR; i++) p[i] = load4(P + (ty + 16 * i) * LDP + k);
#pragma unroll
                    for (int j = 0; j < VJ; j++) {
                        const int c = 4 * vx + 64 * j;
                        if (c >= a.vd) continue;
                        const float4 v0 = load4(V + k * ldv + c), v1 = load4(V + (k + 1) * ldv + c), v2 = load4(V + (k + 2) * ldv + c),
                                     v3 = load4(V + (k + 3) * ldv + c);
#pragma unroll
                        for (int i = 0; i < TR; i++) {
                            add4(o[i][j], p[i].x, v0);
                            add4(o[i][j], p[i].y, v1);
                            add4(o[i][j], p[i].z, v2);
                            add4(o[i][j], p[i].w, v3);
                        }
                    }
                }
            }
            __syncthreads();                     // the stage that the next round fills has been read
        }
        if constexpr (FEW) {                 // the warps' sums, over the stages (4 x 16 rows of values fit them for any sizes)
            if (VJ == 1) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    acc[r][0].x += __shfl_xor_sync(FULL, acc[r][0].x, 16);
                    acc[r][0].y += __shfl_xor_sync(FULL, acc[r][0].y, 16);
                    acc[r][0].z += __shfl_xor_sync(FULL, acc[r][0].z, 16);
                    acc[r][0].w += __shfl_xor_sync(FULL, acc[r][0].w, 16);
                }
            }
            for (int h = 4;; h >>= 1) {          // the last round: warp 0 leaves the result
                __syncthreads();
#pragma unroll
                for (int r = 0; r < 16; r++)
#pragma unroll
                    for (int n = 0; n < NQ; n++)
                        if (warp >= h && warp < max(1, 2 * h) && fc + 128 * n < a.vd) put4(KV + ((warp - h) * 16 + r) * a.vd + fc + 128 * n, acc[r][n]);
                __syncthreads();
                if (h == 0) break;
#pragma unroll
                for (int r = 0; r < 16; r++)
#pragma unroll
                    for (int n = 0; n < NQ; n++)
                        if (warp < h && fc + 128 * n < a.vd) add4(acc[r][n], 1.0f, load4(KV + (warp * 16 + r) * a.vd + fc + 128 * n));
            }
#pragma unroll
            for (int j = 0; j < VJ; j++)
                if (4 * tx + 64 * j < a.vd) o[0][j] = load4(KV + ty * a.vd + 4 * tx + 64 * j);
        }
        float* piece = a.part + ((size_t)blockIdx.x * 2 + it.piece) * tree_piece_floats(RB, a.vd);
        const bool fix = odd != 0;
#pragma unroll
        for (int i = 0; i < TR; i++) {
            const int r = ty + 16 * i, row = s.r0 + min(r, s.rows - 1), node = (int)(row * a.per_magic >> 32);
            const float sum = row_sum(l[i]);
            for (int off = 8; off >= lv; off >>= 1) {
                o[i][0].x += __shfl_xor_sync(FULL, o[i][0].x, off);
                o[i][0].y += __shfl_xor_sync(FULL, o[i][0].y, off);
                o[i][0].z += __shfl_xor_sync(FULL, o[i][0].z, off);
                o[i][0].w += __shfl_xor_sync(FULL, o[i][0].w, off);
            }
            if (r >= s.rows || tx >= lv) continue;
            if (fix)                             // values of attended keys that are not finite (they entered the product as zeros)
                for (int k = max(it.tile, s.edge / TS_KEYS) * TS_KEYS; k < min(s.len + s.n, (it.tile + it.n) * TS_KEYS); k++) {
                    unsigned sees[1];
                    tree_seen<1>(a, s, node, k, sees);
                    if (!(sees[0] & 1u)) continue;
#pragma unroll
                    for (int j = 0; j < VJ; j++) {
                        const int c = 4 * tx + 64 * j;
                        if (c >= a.vd) continue;
                        const float4 x = load4(cache + (size_t)k * a.ld + a.kv_heads * a.kd + it.g * a.vd + c);
                        if (!isfinite(x.x)) o[i][j].x += x.x;
                        if (!isfinite(x.y)) o[i][j].y += x.y;
                        if (!isfinite(x.z)) o[i][j].z += x.z;
                        if (!isfinite(x.w)) o[i][j].w += x.w;
                    }
                }
            if (!it.whole && tx == 0) reinterpret_cast<float2*>(piece)[r] = make_float2(m[i], sum);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // no key seen
            const TreeOut<float> out(a, s.first + node, it.g * a.per_kv + row - node * a.per_kv);
#pragma unroll
            for (int j = 0; j < VJ; j++) {
                const int c = 4 * tx + 64 * j;
                if (c >= a.vd) continue;
                if (it.whole) out.put4at(c, scaled4(o[i][j], inv));
                else put4(piece + 2 * RB + (size_t)r * a.vd + c, o[i][j]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------ pieces
constexpr int TM_WARPS = 8, TM_ML = (2 * TREE_CTAS + 31) / 32;
// grid (X, groups of `per` rows).  With few segments X counts them; else block x looks at the border between the shares of CTAs x and
// x + 1, and when it is the first border inside a segment, the block adds that segment's pieces.  WIDE: the warps of a block share the
// pieces of one row after the other (few rows); else a warp has rows of its own.  HI: values above 128.  Bound by the latency of the
// loads, so what can be is asked for side by side; where the pieces are follows from what the attention kernel has waited for before it
// let this one start.
template <class T, bool WIDE, bool HI>
__global__ void __launch_bounds__(TM_WARPS * 32, 4) k_ftree_merge(const TreeArgs a, int per, int by_segment) {
    __shared__ float4 sum[WIDE ? TM_WARPS : 1][HI ? 64 : 32];
    __shared__ float fac[TM_WARPS][TM_ML * 32];
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long share;
    int cta = blockIdx.x;                                     // the CTA ahead of the border
    TreeShare w;
    if (by_segment) {
        w = tree_start(a, -1, lane, &share, blockIdx.x);
        cta = w.cta;
    } else {
        w = tree_start(a, cta + 1, lane, &share);
    }
    const TreeSeg s = tree_seg(a, w.seg);
    // the border lies at place w.place of the segment
    const int r0 = blockIdx.y * per, r1 = min(s.rows, r0 + per);
    const bool mine = w.left > 0 && tree_tiles(a, s, w.place) > 0 && tree_tiles(a, s, w.place - share) == 0;
    pdl_wait();
    if (!mine || r0 >= r1) return;
    const int behind = tree_places(a, s) - 1 - w.place, n = 2 + (share <= behind ? (int)((unsigned)behind / (unsigned)share) : 0);   // pieces
    const size_t size = tree_piece_floats(a.block, a.vd);
    // the CTA ahead of the border had tiles of the segment before when its share began ahead of this one
    const float* head = a.part + ((size_t)cta * 2 + (w.place < share ? 1 : 0)) * size;
    const float* rest = a.part + (size_t)cta * 2 * size;                      // the others are their CTAs' first pieces
    const int vq = a.vd / 4;
    const bool lo = lane < vq, hi = HI && 32 + lane < vq;
    auto piece = [&](int c) { return c ? rest + c * 2 * size : head; };
    auto finish = [&](int r, float4 o0, float4 o1) {
        const int row = s.r0 + r, node = (int)(row * a.per_magic >> 32);
        const TreeOut<T> out(a, s.first + node, w.g * a.per_kv + row - node * a.per_kv);
        if (lo) out.put4at(lane * 4, o0);
        if (hi) out.put4at(128 + lane * 4, o1);
    };
    if (!WIDE && n <= 4) {                                    // every lane takes all factors of its row
        for (int r = r0 + warp; r < r1; r += TM_WARPS) {
            float2 ml[4];
            float4 x[4], y[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float* p = piece(min(c, n - 1));
                const float* v = p + 2 * a.block + (size_t)r * a.vd + lane * 4;
                ml[c] = c < n ? reinterpret_cast<const float2*>(p)[r] : make_float2(-INFINITY, 0.0f);
                x[c] = lo && c < n ? load4(v) : make_float4(0, 0, 0, 0);
                y[c] = hi && c < n ? load4(v + 128) : make_float4(0, 0, 0, 0);
            }
            float m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), l = 0.0f;
            if (m == -INFINITY) m = 0.0f;                     // a row without keys
            float4 o0 = make_float4(0, 0, 0, 0), o1 = o0;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float f = exp2f(ml[c].x - m);
                l = fmaf(f, ml[c].y, l);
                add4(o0, f, x[c]);
                add4(o1, f, y[c]);
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            finish(r, scaled4(o0, inv), scaled4(o1, inv));
        }
        return;
    }
    for (int r = WIDE ? r0 : r0 + warp; r < r1; r += WIDE ? 1 : TM_WARPS) {
        float2 ml[TM_ML];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < TM_ML; i++) {
            const int c = i * 32 + lane;
            ml[i] = c < n ? reinterpret_cast<const float2*>(piece(c))[r] : make_float2(-INFINITY, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < TM_ML; i++) m = fmaxf(m, ml[i].x);
        m = warp_max(m);
        if (m == -INFINITY) m = 0.0f;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < TM_ML; i++) {
            const float f = exp2f(ml[i].x - m);
            fac[warp][i * 32 + lane] = f;
            l = fmaf(f, ml[i].y, l);
        }
        l = warp_sum(l);
        __syncwarp();
        const size_t at = 2 * a.block + (size_t)r * a.vd + lane * 4;
        float4 o0 = make_float4(0, 0, 0, 0), o1 = o0;
        constexpr int RUN = WIDE || HI ? 4 : 8, STEP = WIDE ? TM_WARPS : 1;
        for (int c0 = WIDE ? warp : 0; c0 < n; c0 += RUN * STEP) {
            float4 x[RUN], y[RUN];
#pragma unroll
            for (int k = 0; k < RUN; k++) {
                const int c = c0 + k * STEP;
                const float* p = piece(c) + at;
                x[k] = lo && c < n ? load4(p) : make_float4(0, 0, 0, 0);
                y[k] = hi && c < n ? load4(p + 128) : make_float4(0, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < RUN; k++) {
                const int c = c0 + k * STEP;
                const float f = c < n ? fac[warp][c] : 0.0f;
                add4(o0, f, x[k]);
                add4(o1, f, y[k]);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (!WIDE) {
            finish(r, scaled4(o0, inv), scaled4(o1, inv));
            continue;
        }
        __syncthreads();
        sum[WIDE ? warp : 0][lane] = o0;
        if (HI) sum[WIDE ? warp : 0][HI ? 32 + lane : 0] = o1;
        __syncthreads();
        if (warp == 0) {
            o0 = o1 = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < (WIDE ? TM_WARPS : 1); i++) {
                add4(o0, inv, sum[i][lane]);
                if (HI) add4(o1, inv, sum[i][HI ? 32 + lane : 0]);
            }
            finish(r, o0, o1);
        }
    }
}

// ------------------------------------------------------------------------------------------------------ host side
constexpr float LOG2_E = 1.4426950408889634f;
template <int TR, int VJ, bool FEW>
static cudaError_t launch_simt(const TreeArgs& a, cudaStream_t q) {
    const size_t smem = simt_smem(a.block, a.kd, a.vd);
    const cudaError_t e = most_smem(k_ftree_simt<TR, VJ, FEW>);
    if (e != cudaSuccess) return e;
    return launch_pdl_try(k_ftree_simt<TR, VJ, FEW>, dim3(a.ctas), dim3(TS_THREADS), smem, q, 1, a);
}
template <int TR, bool FEW>
static cudaError_t launch_simt_v(const TreeArgs& a, cudaStream_t q) {
    return a.vd <= 64 ? launch_simt<TR, 1, FEW>(a, q) : a.vd <= 128 ? launch_simt<TR, 2, FEW>(a, q) : launch_simt<TR, 4, FEW>(a, q);
}
// FEW saves reads of shared memory in every tile and adds the warps' sums in every stretch.  With larger values it is the faster one even at
// two tiles a CTA (8 / 1 heads of 128, two nodes of three sequences behind 2274 keys: 19.8 us, 20.6 without; 21 / 3 heads of 96, a token of four
// sequences behind 22854: 116 / 161), with smaller ones from a few tiles on (8 / 8 heads of 64, 10 tiles: 38.1 / 43.1, 2 tiles: 16.8 / 15.2;
// 4 / 2 heads of 40 and 24, 2 tiles: 14.9 / 11.8).  Values of 24 would want it later still (7 tiles: 27.7 / 22.8).
static bool simt_few(const TreeArgs& a) {
    return a.block == 16 && (a.vd > 64 || (long long)a.seq.seqs * a.kv_heads * a.blocks * (a.seq.max_len / TS_KEYS + 1) >= 6ll * a.ctas);
}
static cudaError_t launch_simt_r(const TreeArgs& a, cudaStream_t q) {
    switch (a.block) {
        case 16: return simt_few(a) ? launch_simt_v<1, true>(a, q) : launch_simt_v<1, false>(a, q);
        case 32: return launch_simt_v<2, false>(a, q);
        case 48: return launch_simt_v<3, false>(a, q);
        default: return launch_simt_v<4, false>(a, q);
    }
}
template <class T>
static cudaError_t launch_merge(const TreeArgs& a, cudaStream_t q) {
    if (a.ctas == 1) return cudaSuccess;
    const long long segs = (long long)a.seq.seqs * a.blocks * a.kv_heads;
    const int by_segment = segs < a.ctas - 1, x = by_segment ? (int)segs : a.ctas - 1, rows = std::min(a.block, a.seq.max_nodes * a.per_kv);
    const bool wide = rows * x <= 4 * TREE_CTAS;              // a row per block, about four blocks on an SM
    const int per = wide ? 1 : TM_WARPS * std::max(1, rows * x / (TM_WARPS * 4 * TREE_CTAS));
    const dim3 grid(x, (rows + per - 1) / per), block(TM_WARPS * 32);
    if (a.vd <= 128)
        return wide ? launch_pdl_try(k_ftree_merge<T, true, false>, grid, block, 0, q, 1, a, per, by_segment)
                    : launch_pdl_try(k_ftree_merge<T, false, false>, grid, block, 0, q, 1, a, per, by_segment);
    return wide ? launch_pdl_try(k_ftree_merge<T, true, true>, grid, block, 0, q, 1, a, per, by_segment)
                : launch_pdl_try(k_ftree_merge<T, false, true>, grid, block, 0, q, 1, a, per, by_segment);
}
// CTAs of an SM: two where registers and shared memory allow it.
static int simt_ctas(const TreeArgs& a) { return a.vd <= 128 && simt_smem(a.block, a.kd, a.vd) <= 112 * 1024 ? 2 : 1; }
// Rows of a block, keys of a tile, tiles that a turn costs.  A tile takes about as long for its copies, waits and softmax as for the
// products of 48 rows.
static void simt_shape(int rows, int* block, int* tile, int* turn) {
    auto cost = [&](int b) { return (long long)((rows + b - 1) / b) * (48 + b); };
    *block = 64;
    for (int b = 48; b >= 16; b -= 16)
        if (cost(b) < cost(*block)) *block = b;
    *tile = TS_KEYS;
    *turn = 1;
}

}  // namespace detb

using namespace detb;

extern "C" {

size_t det_f_tree_scratch_bytes(int heads, int kv_heads, int vdim, int max_nodes) {
    if (heads <= 0 || kv_heads <= 0 || vdim <= 0 || max_nodes <= 0) return 16;
    const int rows = (int)std::min((long long)max_nodes * (heads / kv_heads), 1ll << 24), vd = round8(vdim);
    int block = 0, other = 0, tile = 0, turn = 0;
    simt_shape(rows, &block, &tile, &turn);
    ftree_tc_shape(rows, 8, vd, &other, &tile, &turn);      // the smallest keys have the largest blocks
    block = std::max(2 * block, other);                     // fp32: two CTAs an SM
    return TREE_MAP_BYTES + TREE_CTAS * 2 * tree_piece_floats(block, vd) * sizeof(float);
}

int det_f_tree_attn(const det_ftree_op* op, cudaStream_t st) {
    const char* name = "det_f_tree_attn";
    DETB_TAKE(op != nullptr, "no descriptor");
    DETB_TAKE(op->heads > 0 && op->kv_heads > 0 && op->heads <= 4096 && op->heads % op->kv_heads == 0 && op->dim > 0 && op->vdim > 0 && op->cap > 0,
              "bad sizes");
    DETB_TAKE(op->dim <= 256 && op->vdim <= 256, "the head is too large");
    DETB_TAKE(op->dtype == DET_F32 || op->dtype == DET_BF16, "unknown activation type");
    DETB_TAKE(std::isfinite(op->scale * LOG2_E) && op->scale > 0.0f, "bad scale");
    DETB_TAKE(!op->vrope_cos == !op->vrope_sin && (!op->vrope_cos || (op->vdim % 2 == 0 && op->pos && op->rope_len > 0)), "bad rotation of the values");
    if (const char* why = bad_ref(op->seq)) return refuse(name, why);
    const long long rows = (long long)op->seq.max_nodes * (op->heads / op->kv_heads);
    DETB_TAKE(rows <= 1 << 24 && rows * (op->heads / op->kv_heads) < 1ll << 32, "too many rows");
    DETB_TAKE(!op->mask || (op->seq.max_nodes <= DET_MAX_TREE && op->mask_ld * 32ll >= op->seq.max_nodes), "the mask is too small");
    DETB_TAKE(op->ldo >= op->heads * op->vdim && (!op->gate || op->ldg >= op->heads), "rows overlap");
    if (op->seq.rows == 0 || op->seq.seqs == 0 || rows == 0) return 0;
    DETB_TAKE(op->q && op->out && op->scratch && aligned16(op->q) && reinterpret_cast<uintptr_t>(op->scratch) % 128 == 0,
              "q, out or scratch is NULL or misaligned");
    TreeArgs a{};
    a.heads = op->heads; a.kv_heads = op->kv_heads; a.per_kv = op->heads / op->kv_heads; a.dim = op->dim; a.vdim = op->vdim;
    a.per_magic = ((1ull << 32) + a.per_kv - 1) / a.per_kv;
    a.kd = round8(op->dim); a.vd = round8(op->vdim);
    a.ld = det_f_attn_ld(op->kv_heads, op->dim, op->vdim);
    a.ldq = det_f_attn_q_ld(op->heads, op->dim);
    a.seq = op->seq;
    const bool few = op->dtype == DET_BF16 && ftree_few_takes(a, (int)rows);
    if (few) ftree_few_shape(&a.block, &a.tile);
    else if (op->dtype == DET_BF16) ftree_tc_shape((int)rows, a.kd, a.vd, &a.block, &a.tile, &a.turn);
    else simt_shape((int)rows, &a.block, &a.tile, &a.turn);
    const long long blocks = (rows + a.block - 1) / a.block;
    DETB_TAKE(blocks * op->seq.seqs <= 65535, "too many rows");
    DETB_TAKE(runtime_ready(), "no usable device");
    a.scale2 = op->scale * LOG2_E;
    a.cap = std::min(op->cap, TREE_MAX_KEYS); a.q = op->q; a.mask = op->mask; a.mask_ld = op->mask_ld; a.gate = op->gate; a.ldg = op->ldg; a.pos = op->pos;
    a.rope_len = op->rope_len; a.vcs = op->vrope_cos; a.vsn = op->vrope_sin; a.out = op->out; a.ldo = op->ldo;
    a.maps = op->scratch;
    a.part = reinterpret_cast<float*>(static_cast<char*>(op->scratch) + TREE_MAP_BYTES);
    a.error_flag = error_word();
    a.blocks = (int)blocks;
    a.ctas = std::min(TREE_CTAS, sm_count()) * (op->dtype == DET_F32 ? simt_ctas(a) : 1);
    cudaStream_t q = queue_of(st);
    if (few) return launched(name, ftree_few_launch(a, q));
    if (op->dtype == DET_BF16) {
        if (int rc = launched(name, ftree_tc_launch(a, q))) return rc;
        return launched(name, launch_merge<bf16>(a, q));
    }
    if (int rc = launched(name, launch_simt_r(a, q))) return rc;
    return launched(name, launch_merge<float>(a, q));
}

}  // extern "C"
