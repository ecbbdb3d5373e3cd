// Tree attention over bfloat16 caches for decoded tokens and small trees: 16 query rows of a key/value head are one MMA tile, so a key
// costs 16 rows of products whatever their number, and what bounds the call is the cache's bytes or, for short caches, latency.  One
// launch: a cluster of CTAs shares the keys of a (sequence, key/value head, block of 16 rows), each of its warps walks 16-key tiles
// through a ring of its own, and the cluster adds its pieces over distributed shared memory.
//
// 40 / 8 heads of 128: a token behind 2048 keys 10.5 - 11.4 us (8.4 MB; 129 tiles for the 64 warps of a cluster: a warp walks two or three),
// behind 64 keys 9.0.  So it is the fixed part that it takes: the sequence's place and cache from device memory, the first tiles, one tile's
// products and softmax, two barriers of the cluster and its sum, each waiting for the one before; nearly all of it is the kernel's own time
// (10.0 and 12.5 us from a cold start under ncu).  Tokens of 32 sequences behind 4096 keys 101 us (537 MB, 5.3 TB/s).
#include "flash.cuh"
#include "ftree.cuh"
#include <algorithm>

namespace detb {

constexpr int TF_WARPS = 4, TF_KEYS = 16, TF_STAGES = 3, TF_ROWS = 16;

static size_t few_smem(int kd, int dv) {
    const size_t ldk = ((kd + 15) & ~15) + 8, ring = ((size_t)TF_ROWS * ldk + (size_t)TF_WARPS * TF_STAGES * TF_KEYS * (ldk + dv + 8)) * 2;
    return std::max(ring, (size_t)(TF_WARPS + 1) * TF_ROWS * (dv + 2) * sizeof(float));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned in_cta(unsigned addr, int rank) {       // the same place in another CTA of the cluster
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 far4(unsigned addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 far2(unsigned addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// grid (CTAs of a cluster, key/value heads x row blocks, sequences)
template <int DV>
__global__ void __launch_bounds__(TF_WARPS * 32) k_ftree_few(const TreeArgs a) {
    extern __shared__ __align__(16) uint8_t tfs[];
    __shared__ int odd;                                       // a staged value was not finite
    const int dqp = (a.kd + 15) & ~15, ldk = dqp + 8;
    constexpr int LDV = DV + 8;
    bf16* Q = reinterpret_cast<bf16*>(tfs);                   // [16][ldk]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x, ranks = gridDim.x, g = blockIdx.y / a.blocks, rb = blockIdx.y % a.blocks;
    bf16* Kt = Q + TF_ROWS * ldk + (size_t)warp * TF_STAGES * TF_KEYS * (ldk + LDV);   // this warp's [stage][16][ldk]
    bf16* Vt = Kt + TF_STAGES * TF_KEYS * ldk;                // ... and [stage][16][LDV]
    pdl_trigger();
    if (threadIdx.x == 0) odd = 0;
    if (dqp != a.kd)                                          // what the copies leave unwritten enters products
        for (int i = lane; i < TF_STAGES * TF_KEYS; i += 32) *reinterpret_cast<uint4*>(Kt + i * ldk + a.kd) = make_uint4(0, 0, 0, 0);
    pdl_wait();
    const TreeSeg s = tree_seg(a, blockIdx.z * a.blocks + rb);
    if (s.bad && rank == 0 && blockIdx.y == 0 && threadIdx.x == 0) report_size(a.error_flag);
    if (s.tiles == 0) return;                                 // the whole cluster
    const int per = (s.tiles + ranks - 1) / ranks, t1 = min(s.tiles, (rank + 1) * per);
    const int last = s.len + s.n - 1;
    const bf16* cache = static_cast<const bf16*>(a.seq.table[s.b].cache);
    const int kvec = a.kd / 8, tvec = kvec + a.vd / 8;
    auto fetch = [&](int t, int stage) {
        if (t < t1)
            for (int v = lane; v < tvec; v += 32) {
                const bool val = v >= kvec;
                const bf16* src = cache + (val ? a.kv_heads * a.kd + g * a.vd + (v - kvec) * 8 : g * a.kd + v * 8);
                unsigned dst = smem_addr(val ? Vt + stage * TF_KEYS * LDV + (v - kvec) * 8 : Kt + stage * TF_KEYS * ldk + v * 8);
                const unsigned step = (val ? LDV : ldk) * 2;
#pragma unroll
                for (int k = 0; k < TF_KEYS; k++, dst += step) cp_async16(dst, src + (size_t)min(t * TF_KEYS + k, last) * a.ld);   // past the end: a copy, masked below
            }
        cp_async_commit();
    };
    int t = rank * per + warp;
#pragma unroll
    for (int i = 0; i < TF_STAGES - 1; i++) fetch(t + i * TF_WARPS, i);
    const bf16* q = static_cast<const bf16*>(a.q) + (size_t)s.first * a.ldq + (size_t)g * a.per_kv * a.kd;
    for (int i = threadIdx.x; i < TF_ROWS * (dqp / 8); i += TF_WARPS * 32) {
        const int r = i / (dqp / 8), v = i - r * (dqp / 8), row = s.r0 + r, node = (int)(row * a.per_magic >> 32);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < s.rows && v < kvec) x = *reinterpret_cast<const uint4*>(q + (size_t)node * a.ldq + (row - node * a.per_kv) * a.kd + v * 8);
        *reinterpret_cast<uint4*>(Q + r * ldk + v * 8) = x;
    }
    __syncthreads();
    float o[DV / 8][4];
#pragma unroll
    for (int i = 0; i < DV / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    FlashRows st{{-INFINITY, -INFINITY}, {0.0f, 0.0f}};
    const unsigned qaddr = smem_addr(Q + (lane & 15) * ldk + (lane >> 4) * 8);
    for (int stage = 0; t < t1; t += TF_WARPS, stage = stage + 1 == TF_STAGES ? 0 : stage + 1) {
        fetch(t + (TF_STAGES - 1) * TF_WARPS, stage == 0 ? TF_STAGES - 1 : stage - 1);
        cp_async_wait<TF_STAGES - 1>();
        __syncwarp();
        const int k0 = t * TF_KEYS;
        const bool masked = k0 + TF_KEYS > s.edge;
        bf16* V = Vt + stage * TF_KEYS * LDV;
        if (masked) {                                         // a weight of zero does not undo a value that is not finite
            bool hit = false;
            for (int i = lane; i < TF_KEYS * (a.vd / 2); i += 32) {
                const int k = i / (a.vd / 2);
                unsigned* p = reinterpret_cast<unsigned*>(V + k * LDV) + (i - k * (a.vd / 2));
                unsigned w = *p;
                if (!(((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u)) continue;
                if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
                if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
                *p = w;
                hit = true;
            }
            if (hit) odd = 1;
            __syncwarp();
        }
        float x[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
        const unsigned kaddr = smem_addr(Kt + stage * TF_KEYS * ldk + ((lane & 7) + ((lane >> 4) << 3)) * ldk + ((lane >> 3) & 1) * 8);
#pragma unroll 4
        for (int kk = 0; kk < dqp; kk += 16) {
            unsigned qa[4], kb[4];
            ldsm4(qaddr + kk * 2, qa);
            ldsm4(kaddr + kk * 2, kb);
            mma16816(x[0], qa, kb[0], kb[1]);
            mma16816(x[1], qa, kb[2], kb[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) x[n][c] *= a.scale2;
        if (masked) {
            unsigned seen[2][1];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = s.r0 + min((lane >> 2) + i * 8, s.rows - 1);
                tree_seen<1>(a, s, (int)(row * a.per_magic >> 32), k0, seen[i]);
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (!((seen[c >> 1][0] >> (n * 8 + (lane & 3) * 2 + (c & 1))) & 1u)) x[n][c] = -INFINITY;
            __syncwarp();
        }
        unsigned pf[1][4];
        flash_softmax(st, x, o, pf);
        const unsigned vaddr = smem_addr(V + (lane & 15) * LDV + (lane >> 4) * 8);
#pragma unroll
        for (int n = 0; n < DV / 16; n++) {
            unsigned vb[4];
            ldsm4_t(vaddr + n * 32, vb);
            mma16816(o[2 * n], pf[0], vb[0], vb[1]);
            mma16816(o[2 * n + 1], pf[0], vb[2], vb[3]);
        }
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();
    // the warps' pieces: [warp][row][DV] values, then [warp][row] maximum and sum; behind them the CTA's
    float* po = reinterpret_cast<float*>(tfs);
    float* ml = po + TF_WARPS * TF_ROWS * DV;
    float* mine = ml + TF_WARPS * TF_ROWS * 2;                // [row][DV], then [row] maximum and sum
    float* mine_ml = mine + TF_ROWS * DV;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        st.l[i] += __shfl_xor_sync(FULL, st.l[i], 1);
        st.l[i] += __shfl_xor_sync(FULL, st.l[i], 2);
        const int at = warp * TF_ROWS + (lane >> 2) + i * 8;
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + at * 2) = make_float2(st.m[i], st.l[i]);
#pragma unroll
        for (int n = 0; n < DV / 8; n++)
            *reinterpret_cast<float2*>(po + (size_t)at * DV + n * 8 + (lane & 3) * 2) = make_float2(o[n][i * 2], o[n][i * 2 + 1]);
    }
    __syncthreads();
    const int vq = a.vd / 4, items = s.rows * vq;
    for (int i = threadIdx.x; i < items; i += TF_WARPS * 32) {
        const int r = i / vq, v = (i - r * vq) * 4;
        float m = -INFINITY, l = 0.0f;
        float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < TF_WARPS; w++) m = fmaxf(m, ml[(w * TF_ROWS + r) * 2]);
        const float base = m == -INFINITY ? 0.0f : m;         // no key seen
#pragma unroll
        for (int w = 0; w < TF_WARPS; w++) {
            const int at = w * TF_ROWS + r;
            const float f = exp2f(ml[at * 2] - base);
            l = fmaf(f, ml[at * 2 + 1], l);
            add4(y, f, *reinterpret_cast<const float4*>(po + (size_t)at * DV + v));
        }
        put4(mine + r * DV + v, y);
        if (v == 0) *reinterpret_cast<float2*>(mine_ml + r * 2) = make_float2(m, l);
    }
    __syncwarp();
    cluster_sync();
    // the cluster's: every CTA adds its share of the rows' values
    const unsigned far = smem_addr(mine), far_ml = smem_addr(mine_ml), far_odd = smem_addr(&odd);
    for (int i = rank * TF_WARPS * 32 + threadIdx.x; i < items; i += ranks * TF_WARPS * 32) {
        const int r = i / vq, v = (i - r * vq) * 4;
        float m = -INFINITY, l = 0.0f;
        float4 y = make_float4(0, 0, 0, 0);
        bool fix = false;
#pragma unroll 8
        for (int c = 0; c < ranks; c++) m = fmaxf(m, far2(in_cta(far_ml + r * 8, c)).x);
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll 8
        for (int c = 0; c < ranks; c++) {
            const float2 x = far2(in_cta(far_ml + r * 8, c));
            const float f = exp2f(x.x - base);
            l = fmaf(f, x.y, l);
            add4(y, f, far4(in_cta(far + (r * DV + v) * 4, c)));
            int any;
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(any) : "r"(in_cta(far_odd, c)) : "memory");
            fix |= any != 0;
        }
        const int row = s.r0 + r, node = (int)(row * a.per_magic >> 32);
        y = scaled4(y, l == 0.0f ? 0.0f : 1.0f / l);
        if (fix) {                                            // values of attended keys that are not finite (they entered the product as zeros)
            float z[4] = {y.x, y.y, y.z, y.w};
            for (int k = s.edge / TF_KEYS * TF_KEYS; k <= last; k++) {
                unsigned sees[1];
                tree_seen<1>(a, s, node, k, sees);
                if (!(sees[0] & 1u)) continue;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = to_f(cache[(size_t)k * a.ld + a.kv_heads * a.kd + g * a.vd + v + j]);
                    if (!isfinite(x)) z[j] += x;
                }
            }
            y = make_float4(z[0], z[1], z[2], z[3]);
        }
        TreeOut<bf16>(a, s.first + node, g * a.per_kv + row - node * a.per_kv).put4at(v, y);
    }
    __syncwarp();
    cluster_sync();                                           // nobody leaves while its pieces are read
}

template <int DV>
static cudaError_t launch(const TreeArgs& a, int ranks, cudaStream_t q) {
    const size_t smem = few_smem(a.kd, DV);
    cudaError_t e = most_smem(k_ftree_few<DV>);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_ftree_few<DV>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    return launch_pdl_try(k_ftree_few<DV>, dim3(ranks, a.kv_heads * a.blocks, a.seq.seqs), dim3(TF_WARPS * 32), smem, q, ranks, a);
}

// CTAs of a cluster: a power of two, so that all clusters fill the device about twice over, and no more than there are tiles for the
// warps.  Clusters of 16 find room eight at a time (16 of them took two rounds: 20.4 us where 24 clusters of 8 took 11.1).
static int few_ranks(long long clusters, int max_len) {
    const int tiles = max_len / TF_KEYS + 1;
    int ranks = 1;
    while (ranks < (clusters <= 8 ? 16 : 8) && clusters * ranks * 2 <= 2 * TREE_CTAS && ranks * TF_WARPS < tiles) ranks *= 2;
    return ranks;
}
// This kernel or k_ftree_tc, by what both were measured to take (in us, 8 key/value heads of 128, this one / the other):
//   here   8.5 for every round of CTAs, and the cache's bytes once per 16 rows at 24 GB/s a CTA (keys and values of 128 in its ring; 32 for
//          larger ones, 33 / 23 at 64 rows of 4096 keys of 256), 6 TB/s together: 11.3 / 16.9 at 5 rows of 512 keys, 14.3 / 20.1 at 40
//          rows of 2048, 30.4 / 24.1 at 40 rows of 8192, 48 / 41 at 5 rows of 32768; 95 / 109 for 4 sequences of those; 32 / 41 for 16
//          sequences of 2048 keys and 5 rows, 98 / 45 with 40 rows
//   there  15 for its start and its second launch, 5 for a turn, the larger of the bytes at 5.8 TB/s and 1.45 for a tile of 128 x 128
bool ftree_few_takes(const TreeArgs& a, int rows) {
    const int blocks = (rows + TF_ROWS - 1) / TF_ROWS;
    const long long clusters = (long long)a.seq.seqs * a.kv_heads * blocks, len = (long long)a.seq.max_len + a.seq.max_nodes;
    if (blocks > 16 || (long long)a.kv_heads * blocks > 65535 || (float_flags() & 16)) return false;
    if (float_flags() & 32) return true;
    const int dv = a.vd <= 64 ? 64 : a.vd <= 128 ? 128 : 256;
    const double row = 2.0 * (a.kd + a.vd), heads = (double)a.kv_heads * a.seq.seqs, bytes = row * heads * (double)len;
    const double slots = (few_smem(a.kd, dv) <= 113 * 1024 ? 2.0 : 1.0) * TREE_CTAS, ctas = (double)clusters * few_ranks(clusters, a.seq.max_len);
    const double here = 8.5e-6 * (double)((long long)(ctas / slots + 0.999)) + bytes * blocks / std::min(std::min(ctas, slots) * std::min(24e9 * row / 512, 32e9), 6e12);
    const double tiles = heads * (double)(len / 128 + 1) * ((rows + 127) / 128);
    const double there = 15e-6 + heads / TREE_CTAS * 5e-6 + std::max(bytes / 5.8e12, tiles / TREE_CTAS * 1.45e-6);
    return here <= there;
}
void ftree_few_shape(int* block, int* tile) {
    *block = TF_ROWS;
    *tile = TF_KEYS;
}
cudaError_t ftree_few_launch(const TreeArgs& a, cudaStream_t q) {
    const int ranks = few_ranks((long long)a.seq.seqs * a.kv_heads * a.blocks, a.seq.max_len);
    return a.vd <= 64 ? launch<64>(a, ranks, q) : a.vd <= 128 ? launch<128>(a, ranks, q) : launch<256>(a, ranks, q);
}

}  // namespace detb
