// Position rotation (include/det_b200.h): tables of cosines and sines with the scalings for long contexts, and the pass that
// norms, rotates and caches the rows of a step.
//
//   k_frope_table   a thread owns up to four neighbouring columns and walks down the positions.
//   k_fqk_rope      a warp takes some heads of a row, one per 8 to 32 lanes at a time.
#include "ftree.cuh"
#include <algorithm>
#include <cmath>

namespace detb {

// ------------------------------------------------------------------------------------------------------ tables
struct RopeArgs {
    int cols, n, pos0, scaling;
    double log2_base, dims, inv_factor, turns0, low, inv_span;   // turns0: positions / 2 pi within orig_ctx
    float mscale;
    float* cs;
    float* sn;
};
// Turns per position of column i.  In units u = 2^-53: log2 of the base is off by 2 u of itself (with a scaled base the sum by 5 u of its terms),
// the quotient and the product by one each, so f by ln 2 * (4 or 7) u * g, g the size of the exponent; exp2 adds 2 u, 1 / 2 pi and its product 2,
// the linear factor 2: together below (5 g + 9) u.  The ramp's weight is off by (2.8 g + 9) u of (weight + low / span), which the factor between
// both ends of the ramp scales.
__device__ __forceinline__ double turns_of(const RopeArgs& a, int i) {
    constexpr double INV_2PI = 0.15915494309189533577;
    const double f = exp2(-2.0 * i / a.dims * a.log2_base);
    double t = f * INV_2PI;
    if (a.scaling == DET_ROPE_LINEAR) t *= a.inv_factor;
    if (a.scaling == DET_ROPE_RAMP) {
        const double w = fmin(fmax((a.turns0 * f - a.low) * a.inv_span, 0.0), 1.0);
        t *= w + (1.0 - w) * a.inv_factor;
    }
    return t;
}
// cos and sin of `phase` / 2^32 turns.  The quadrant is an integer, what is left (an eighth of a turn either way) goes through the Taylor
// series of both functions, r^11 and r^12 the first terms left out (4e-9 and 1e-10 of the result).
__device__ __forceinline__ float2 turn(unsigned phase, float m) {
    const unsigned q = (phase + 0x20000000u) >> 30;
    const float r = (float)(int)(phase - (q << 30)) * 1.46291807926715968e-9f, x = r * r;      // 2 pi / 2^32
    float s = fmaf(x, 2.75573192e-6f, -1.98412698e-4f);
    s = fmaf(s, x, 8.33333333e-3f);
    s = fmaf(s, x, -1.66666667e-1f);
    s = fmaf(s * x, r, r);
    float c = fmaf(x, -2.75573192e-7f, 2.48015873e-5f);
    c = fmaf(c, x, -1.38888889e-3f);
    c = fmaf(c, x, 4.16666667e-2f);
    c = fmaf(c, x, -0.5f);
    c = fmaf(c, x, 1.0f);
    const float u = q & 1 ? s : c, v = q & 1 ? c : s;
    // cos: - in quadrants 1 and 2; sin: - in quadrants 2 and 3
    return make_float2(__uint_as_float(__float_as_uint(u) ^ ((q + 1) >> 1 << 31)) * m, __uint_as_float(__float_as_uint(v) ^ (q >> 1 << 31)) * m);
}
// One more turn is no turn: a column's turns per position are kept as 64 bits behind the point, and a position's phase is the product's
// low 64 bits, of which the upper half is used (2^-32 turns).  Products of binary64 in its place are what the call took longest over:
// 262144 x 64 pairs took 38.4 us, now 23.2 (134 MB written, 5.8 TB/s: bound by the stores).
template <int V>
__global__ void __launch_bounds__(256) k_frope_table(const RopeArgs a) {
    pdl_trigger();
    const int groups = a.cols / V, g = blockIdx.x * blockDim.x + threadIdx.x;
    unsigned long long t[V];
    if (g < groups)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const double x = turns_of(a, g * V + j);
            t[j] = __double2ull_rn((x - floor(x)) * 18446744073709551616.0);
        }
    pdl_wait();
    if (g >= groups) return;
    for (unsigned p = blockIdx.y * blockDim.y + threadIdx.y; p < (unsigned)a.n; p += gridDim.y * blockDim.y) {      // n fits 31 bits, the sum 32
        const unsigned at = (unsigned)a.pos0 + p;
        float c[V], s[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float2 v = turn((unsigned)(at * t[j] >> 32), a.mscale);
            c[j] = v.x;
            s[j] = v.y;
        }
        const size_t to = (size_t)p * a.cols + (size_t)g * V;
        if (V == 4) {
            *reinterpret_cast<float4*>(a.cs + to) = make_float4(c[0], c[V > 1], c[V > 2 ? 2 : 0], c[V > 3 ? 3 : 0]);
            *reinterpret_cast<float4*>(a.sn + to) = make_float4(s[0], s[V > 1], s[V > 2 ? 2 : 0], s[V > 3 ? 3 : 0]);
        } else {
            a.cs[to] = c[0];
            a.sn[to] = s[0];
        }
    }
}

// ------------------------------------------------------------------------------------------------------ norm and rotation
struct QkArgs {
    int heads, kv_heads, dim, vdim, rot, half, kd, vd, ld, ldq, cap, ldy, q_off, k_off, v_off, rope_len;
    float eps;
    const float* q_norm;
    const float* k_norm;
    const float* y;
    const float* cs;
    const float* sn;
    const float* vcs;
    const float* vsn;
    const int* pos;
    void* q;
    int* error_flag;
    det_tree_ref seq;
};
// n elements from e on (8 of them, zeros past the end).
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int e, int n, float (&v)[8]) {
    if (VEC) {
        const float4 a = e < n ? *reinterpret_cast<const float4*>(p + e) : make_float4(0, 0, 0, 0);
        const float4 b = e < n ? *reinterpret_cast<const float4*>(p + e + 4) : make_float4(0, 0, 0, 0);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = e + i < n ? p[e + i] : 0.0f;
    }
}
__device__ __forceinline__ void put8(float* p, const float (&v)[8]) {
    put4(p, make_float4(v[0], v[1], v[2], v[3]));
    put4(p + 4, make_float4(v[4], v[5], v[6], v[7]));
}
__device__ __forceinline__ void put8(bf16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf(v[0], v[1]), pack_bf(v[2], v[3]), pack_bf(v[4], v[5]), pack_bf(v[6], v[7]));
}

// One pass, bound by HBM: 8192 rows of 40 / 8 heads of 128 into bfloat16 take 70-73 us (357 MB, 5.0 TB/s), in fp32 85 us (474 MB, 5.6 TB/s);
// a single row 3.2 us, the latency of place, row and tables one after the other.  Without VEC: heads of 124 137 us (2.5 TB/s, bound by loads
// and table reads of four bytes), heads of 128 with 24 elements rotated in pairs 83 us.
//
// A warp takes a part of a row's heads, 32 / LPH at a time, eight neighbouring elements a lane; the row's place, its cosines and sines and
// the norm's weights are fetched once.  VEC: heads are multiples of 8 elements, everything is 16-byte aligned and the halves of a
// rotated head are whole lanes apart, so that a lane gets its partners by a shuffle.
constexpr int QK_THREADS = 256;
struct QkLane {
    int e, first, from;            // element, in the first half of the pairs, the lane with the partners
    float co[8], si[8];            // of four pairs, or of eight elements of a half (si with the sign of its product)
};
// `count` heads of n elements from x on, results to `to`: normed by w (or NULL), rotated in the first `rot` elements (or 0).
template <class T, bool VEC, int LPH>
__device__ __forceinline__ void qk_heads(const QkArgs& a, const QkLane& k, const float* x, T* to, int count, int n, int nd, const float* w, int rot, bool half,
                                         size_t pos, int part, int parts) {
    constexpr int HEADS = 32 / LPH;
    const int lane = threadIdx.x & 31, hr = rot / 2;
    float g[8];
    if (w) load8<VEC>(w, k.e, n, g);
    const float inv_n = 1.0f / (float)n;
    int h = part * HEADS + lane / LPH;
    x += h * n;
    to += h * nd + k.e;
    const int left = (count - part * HEADS + parts * HEADS - 1) / (parts * HEADS);       // rounds of the warp
    float ahead[8];
    load8<VEC>(x, k.e, h < count ? n : 0, ahead);
    for (int i = 0; i < left; i++) {
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = ahead[j];
        const float* mine = x;
        const bool real = h < count;
        h += parts * HEADS;
        x += parts * HEADS * n;
        if (i + 1 < left) load8<VEC>(x, k.e, h < count ? n : 0, ahead);
        float r = 1.0f;
        if (w) {
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                s0 = fmaf(z[j], z[j], s0);
                s1 = fmaf(z[j + 1], z[j + 1], s1);
            }
            s0 += s1;
#pragma unroll
            for (int off = LPH / 2; off > 0; off >>= 1) s0 += __shfl_xor_sync(FULL, s0, off);
            r = rsqrtf(fmaf(s0, inv_n, a.eps));
#pragma unroll
            for (int j = 0; j < 8; j++) z[j] *= r * g[j];
        }
        if (rot && half && VEC) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float p = __shfl_sync(FULL, z[j], k.from);
                if (k.e < rot) z[j] = fmaf(z[j], k.co[j], p * k.si[j]);
            }
        } else if (rot && half) {
            // the other half of the pairs comes from memory again (the lines are in L1) and is normed here too
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (real && k.e + j < rot) {
                    const bool first = k.e + j < hr;
                    const int i0 = first ? k.e + j : k.e + j - hr, o = first ? k.e + j + hr : i0;
                    float p = mine[o];
                    if (w) p *= r * w[o];
                    z[j] = fmaf(z[j], a.cs[pos * hr + i0], (first ? -p : p) * a.sn[pos * hr + i0]);
                }
        } else if (rot) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k.e + 2 * j < rot) {
                    const float p = z[2 * j];
                    z[2 * j] = fmaf(p, k.co[j], -(z[2 * j + 1] * k.si[j]));
                    z[2 * j + 1] = fmaf(z[2 * j + 1], k.co[j], p * k.si[j]);
                }
        }
        if (real && k.e < nd) put8(to, z);
        to += parts * HEADS * nd;
    }
}
template <bool VEC, int LPH>
__device__ __forceinline__ QkLane qk_lane(const float* cs, const float* sn, size_t pos, int rot, bool half) {
    QkLane k;
    const int lane = threadIdx.x & 31, l = lane % LPH, hr = rot / 2;
    k.e = l * 8;
    k.first = k.e < hr;
    k.from = lane - l + ((l + (k.first ? hr / 8 : LPH - hr / 8)) & (LPH - 1));
#pragma unroll
    for (int i = 0; i < 8; i++) k.co[i] = 1.0f, k.si[i] = 0.0f;
    if (k.e >= rot) return k;
    cs += pos * hr;
    sn += pos * hr;
    if (half && VEC) {
        load8<VEC>(cs, k.first ? k.e : k.e - hr, hr, k.co);
        load8<VEC>(sn, k.first ? k.e : k.e - hr, hr, k.si);
        if (k.first)
#pragma unroll
            for (int i = 0; i < 8; i++) k.si[i] = -k.si[i];
    } else if (!half) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (k.e / 2 + i < hr) {
                k.co[i] = cs[k.e / 2 + i];
                k.si[i] = sn[k.e / 2 + i];
            }
    }
    return k;
}
// The last block looks through the sequences and reports those that do not fit (of which the buffers may hold no row); the others take the
// rows.  What a sequence's verdict costs a single row: 3.11 -> 3.21 us (one by the row alone -> by its sequence; as the first block 3.25).
template <class T, bool VEC, int LPH>
__global__ void __launch_bounds__(QK_THREADS, 4) k_fqk_rope(const QkArgs a, int parts) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x == gridDim.x - 1) {
        bool bad = false;
        for (int b = threadIdx.x; b < a.seq.seqs; b += QK_THREADS) bad |= tree_span(a.seq, a.cap, b).bad;
        if (bad) report_size(a.error_flag);
        return;
    }
    const int lane = threadIdx.x & 31, task = (int)(((long long)blockIdx.x * QK_THREADS + threadIdx.x) >> 5), row = task / parts, part = task - row * parts;
    if (row >= a.seq.rows) return;
    const TreePlace at = tree_place(a.seq, a.cap, row, lane);
    if (at.nobodys) return;
    const int pos = a.pos ? a.pos[row] : at.slot;
    if (at.slot < 0 || ((a.rot || a.vcs) && (pos < 0 || pos >= a.rope_len))) {
        if (lane == 0) report_size(a.error_flag);
        return;
    }
    const float* y = a.y + (size_t)row * a.ldy;
    T* cache = static_cast<T*>(at.cache) + (size_t)at.slot * a.ld;
    // a group of heads after the other goes round the warps of the row: queries, then keys, then values
    constexpr int HEADS = 32 / LPH;
    const int gq = (a.heads + HEADS - 1) / HEADS, gk = (a.kv_heads + HEADS - 1) / HEADS;
    const int pk = (part + parts - gq % parts) % parts, pv = (pk + parts - gk % parts) % parts;
    const QkLane k = qk_lane<VEC, LPH>(a.cs, a.sn, pos, a.rot, a.half);
    qk_heads<T, VEC, LPH>(a, k, y + a.q_off, static_cast<T*>(a.q) + (size_t)row * a.ldq, a.heads, a.dim, a.kd, a.q_norm, a.rot, a.half, pos, part, parts);
    qk_heads<T, VEC, LPH>(a, k, y + a.k_off, cache, a.kv_heads, a.dim, a.kd, a.k_norm, a.rot, a.half, pos, pk, parts);
    cache += a.kv_heads * a.kd;
    if (a.vcs)
        qk_heads<T, VEC, LPH>(a, qk_lane<VEC, LPH>(a.vcs, a.vsn, pos, a.vdim, false), y + a.v_off, cache, a.kv_heads, a.vdim, a.vd, nullptr, a.vdim, false, pos, pv,
                              parts);
    else qk_heads<T, VEC, LPH>(a, k, y + a.v_off, cache, a.kv_heads, a.vdim, a.vd, nullptr, 0, false, pos, pv, parts);
}

template <class T, bool VEC>
static cudaError_t launch_qk(const QkArgs& a, cudaStream_t q) {
    const int most = std::max(a.kd, a.vd), lph = most <= 64 ? 8 : most <= 128 ? 16 : 32, groups = (a.heads + 2 * a.kv_heads + 32 / lph - 1) / (32 / lph);
    // a group per warp while that leaves SMs idle, fourteen in long runs (8192 rows of 40/8 x 128: 87 us with four, 74 with seven, 70)
    const int parts = (int)std::max<long long>((groups + 13) / 14, std::min<long long>(groups, 32ll * sm_count() / a.seq.rows));
    const long long warps = (long long)a.seq.rows * parts;
    const dim3 grid((unsigned)((warps + QK_THREADS / 32 - 1) / (QK_THREADS / 32) + 1)), block(QK_THREADS);
    return lph == 8    ? launch_pdl_try(k_fqk_rope<T, VEC, 8>, grid, block, 0, q, 1, a, parts)
           : lph == 16 ? launch_pdl_try(k_fqk_rope<T, VEC, 16>, grid, block, 0, q, 1, a, parts)
                       : launch_pdl_try(k_fqk_rope<T, VEC, 32>, grid, block, 0, q, 1, a, parts);
}

}  // namespace detb

using namespace detb;

extern "C" {

int det_f_rope_table(const det_frope_op* op, cudaStream_t st) {
    const char* name = "det_f_rope_table";
    DETB_TAKE(op != nullptr, "no descriptor");
    DETB_TAKE(op->dims >= 2 && op->dims % 2 == 0 && op->n >= 0 && op->pos0 >= 0, "bad sizes");
    DETB_TAKE((long long)op->pos0 + op->n <= 0x7fffffffll, "positions beyond 31 bits");
    DETB_TAKE(std::isfinite(op->base) && op->base > 0.0 && std::isfinite(op->mscale), "bad base or mscale");
    DETB_TAKE(op->scaling >= DET_ROPE_PLAIN && op->scaling <= DET_ROPE_RAMP, "unknown scaling");
    const bool scaled = op->scaling != DET_ROPE_PLAIN, ramp = op->scaling == DET_ROPE_RAMP;
    DETB_TAKE(!scaled || (std::isfinite(op->factor) && op->factor > 0.0), "bad factor");
    DETB_TAKE(op->scaling != DET_ROPE_BASE || op->dims > 2, "the base cannot be scaled for two dimensions");
    DETB_TAKE(!ramp || (std::isfinite(op->orig_ctx) && op->orig_ctx > 0.0 && std::isfinite(op->low) && std::isfinite(op->high) && op->high > op->low),
              "bad ramp");
    if (op->n == 0) return 0;
    DETB_TAKE(op->cos && op->sin, "no tables");
    DETB_TAKE(runtime_ready(), "no usable device");
    RopeArgs a{};
    a.cols = op->dims / 2;
    a.n = op->n;
    a.pos0 = op->pos0;
    a.scaling = op->scaling;
    a.dims = op->dims;
    a.log2_base = std::log2(op->base);
    if (op->scaling == DET_ROPE_BASE) a.log2_base += std::log2(op->factor) * a.dims / (a.dims - 2.0);
    a.inv_factor = scaled ? 1.0 / op->factor : 1.0;
    if (ramp) {
        a.turns0 = op->orig_ctx / 6.283185307179586477;
        a.low = op->low;
        a.inv_span = 1.0 / (op->high - op->low);
    }
    a.mscale = op->mscale;
    a.cs = op->cos;
    a.sn = op->sin;
    const bool four = a.cols % 4 == 0 && aligned16(op->cos) && aligned16(op->sin);
    const int groups = four ? a.cols / 4 : a.cols;
    int tx = 1;
    while (tx < groups && tx < 32) tx *= 2;
    const dim3 block(tx, 256 / tx);
    const int gx = (groups + tx - 1) / tx, want = std::max(1, 8 * sm_count() / gx);
    const dim3 grid(gx, std::min(want, (a.n - 1) / (int)block.y + 1));
    cudaStream_t q = queue_of(st);
    return launched(name, four ? launch_pdl_try(k_frope_table<4>, grid, block, 0, q, 1, a) : launch_pdl_try(k_frope_table<1>, grid, block, 0, q, 1, a));
}

int det_f_qk_rope(const det_fqk_op* op, cudaStream_t st) {
    const char* name = "det_f_qk_rope";
    DETB_TAKE(op != nullptr, "no descriptor");
    DETB_TAKE(op->heads > 0 && op->kv_heads > 0 && op->heads <= 4096 && op->kv_heads <= 4096 && op->dim > 0 && op->vdim > 0 && op->cap > 0,
              "bad sizes");
    DETB_TAKE(op->dim <= 256 && op->vdim <= 256, "the head is too large");
    DETB_TAKE(op->dtype == DET_F32 || op->dtype == DET_BF16, "unknown activation type");
    DETB_TAKE(op->rot_dims >= 0 && op->rot_dims % 2 == 0 && op->rot_dims <= op->dim && (op->half == 0 || op->half == 1), "bad rotation");
    DETB_TAKE(!op->vrope_cos == !op->vrope_sin && (!op->vrope_cos || op->vdim % 2 == 0), "bad rotation of the values");
    DETB_TAKE(op->q_off >= 0 && op->k_off >= 0 && op->v_off >= 0 && op->ldy >= 0, "bad columns");
    DETB_TAKE(std::isfinite(op->eps) && op->eps >= 0.0f, "bad eps");
    if (const char* why = bad_ref(op->seq)) return refuse(name, why);
    if (op->seq.rows == 0 || op->seq.seqs == 0 || op->seq.max_nodes == 0) return 0;
    DETB_TAKE(op->y && op->q && aligned16(op->q), "y or q is NULL or misaligned");
    DETB_TAKE(!op->rot_dims || (op->rope_cos && op->rope_sin), "no tables");
    DETB_TAKE((!op->rot_dims && !op->vrope_cos) || op->rope_len > 0, "empty tables");
    DETB_TAKE(runtime_ready(), "no usable device");
    QkArgs a{};
    a.heads = op->heads; a.kv_heads = op->kv_heads; a.dim = op->dim; a.vdim = op->vdim; a.rot = op->rot_dims; a.half = op->half;
    a.kd = round8(op->dim); a.vd = round8(op->vdim);
    a.ld = det_f_attn_ld(op->kv_heads, op->dim, op->vdim);
    a.ldq = det_f_attn_q_ld(op->heads, op->dim);
    a.cap = op->cap; a.ldy = op->ldy; a.q_off = op->q_off; a.k_off = op->k_off; a.v_off = op->v_off; a.rope_len = op->rope_len;
    a.eps = op->eps; a.q_norm = op->q_norm; a.k_norm = op->k_norm; a.y = op->y;
    a.cs = op->rope_cos; a.sn = op->rope_sin; a.vcs = op->vrope_cos; a.vsn = op->vrope_sin;
    a.pos = op->pos; a.q = op->q; a.error_flag = error_word(); a.seq = op->seq;
    DETB_TAKE((long long)op->seq.rows * (a.heads + 2 * a.kv_heads) < 1ll << 31, "too many rows");
    const bool vec = aligned16(op->y) && op->ldy % 4 == 0 && op->q_off % 4 == 0 && op->k_off % 4 == 0 && op->v_off % 4 == 0 && op->dim % 8 == 0 &&
                     op->vdim % 8 == 0 && aligned16(op->q_norm) && aligned16(op->k_norm) && op->rot_dims % 16 == 0 && aligned16(op->rope_cos) &&
                     aligned16(op->rope_sin);
    cudaStream_t q = queue_of(st);
    cudaError_t e;
    if (op->dtype == DET_BF16) e = vec ? launch_qk<bf16, true>(a, q) : launch_qk<bf16, false>(a, q);
    else e = vec ? launch_qk<float, true>(a, q) : launch_qk<float, false>(a, q);
    return launched(name, e);
}

}  // extern "C"
