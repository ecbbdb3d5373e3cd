// Position rotation (include/det_b200.h): tables of cosines and sines with the scalings for long contexts, and the pass that
// norms, rotates and caches the rows of a step.
//
//   k_frope_table   a thread owns up to four neighbouring columns and walks down the positions.
//   k_fqk_rope      one head of a row per group of 8 to 32 lanes.
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
// Turns per position of column i.
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
// cos and sin of 2 pi x: whole turns leave in binary64, what is left is taken in two fp32 parts, the small one to first order.
__device__ __forceinline__ float2 turn(double x, float m) {
    const double r = 2.0 * (x - rint(x));
    const float hi = (float)r, lo = (float)(r - (double)hi) * 3.14159265f;
    float s, c;
    sincospif(hi, &s, &c);
    return make_float2(fmaf(-lo, s, c) * m, fmaf(lo, c, s) * m);
}
template <int V>
__global__ void __launch_bounds__(256) k_frope_table(const RopeArgs a) {
    pdl_trigger();
    const int groups = a.cols / V, g = blockIdx.x * blockDim.x + threadIdx.x;
    double t[V];
    if (g < groups)
#pragma unroll
        for (int j = 0; j < V; j++) t[j] = turns_of(a, g * V + j);
    pdl_wait();
    if (g >= groups) return;
    for (int p = blockIdx.y * blockDim.y + threadIdx.y; p < a.n; p += gridDim.y * blockDim.y) {
        const double at = (double)a.pos0 + (double)p;
        float c[V], s[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float2 v = turn(at * t[j], a.mscale);
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
    int heads, kv_heads, dim, vdim, rot, half, kd, vd, ld, ldq, cap, ldy, q_off, k_off, v_off, rope_len, lanes;
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
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int e, int n) {
    if (VEC) return e < n ? *reinterpret_cast<const float4*>(p + e) : make_float4(0, 0, 0, 0);
    return make_float4(e < n ? p[e] : 0.0f, e + 1 < n ? p[e + 1] : 0.0f, e + 2 < n ? p[e + 2] : 0.0f, e + 3 < n ? p[e + 3] : 0.0f);
}

constexpr int QK_THREADS = 256;
// grid (rows, pieces of a row's heads); `lanes` lanes per head, four neighbouring elements each, CH times.
template <class T, bool VEC, int CH>
__global__ void __launch_bounds__(QK_THREADS) k_fqk_rope(const QkArgs a) {
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x, lane = threadIdx.x & 31;
    const TreePlace at = tree_place(a.seq, row, lane);
    if (at.b < 0) return;
    const int pos = a.pos ? a.pos[row] : at.slot;
    void* base = a.seq.table[at.b].cache;
    if (at.node < 0 || at.node >= a.seq.max_nodes || at.slot < at.node || at.slot >= a.cap || !usable_cache(base) ||
        ((a.rot || a.vcs) && (pos < 0 || pos >= a.rope_len))) {
        if (threadIdx.x == 0) report_size(a.error_flag);
        return;
    }
    const int u = (blockIdx.y * QK_THREADS + threadIdx.x) / a.lanes, l = threadIdx.x % a.lanes;
    const int units = a.heads + 2 * a.kv_heads;
    const bool value = u >= a.heads + a.kv_heads, key = !value && u >= a.heads;
    const int h = value ? u - a.heads - a.kv_heads : key ? u - a.heads : u;
    const int n = value ? a.vdim : a.dim, nd = value ? a.vd : a.kd;
    const float* x = a.y + (size_t)row * a.ldy + (value ? a.v_off : key ? a.k_off : a.q_off) + (size_t)h * n;
    const float* w = value ? nullptr : key ? a.k_norm : a.q_norm;
    float4 v[CH];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        v[c] = u < units ? load4<VEC>(x, (c * 32 + l) * 4, n) : make_float4(0, 0, 0, 0);
        sum = fmaf(v[c].x, v[c].x, fmaf(v[c].y, v[c].y, fmaf(v[c].z, v[c].z, fmaf(v[c].w, v[c].w, sum))));
    }
    for (int off = a.lanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
    if (u >= units) return;
    const float r = w ? 1.0f / sqrtf(sum / (float)n + a.eps) : 1.0f;
    const int rot = value ? (a.vcs ? a.vdim : 0) : a.rot, half = value ? 0 : a.half, hr = rot / 2;
    const float* cs = (value ? a.vcs : a.cs) + (size_t)pos * hr;
    const float* sn = (value ? a.vsn : a.sn) + (size_t)pos * hr;
    T* to;
    if (value || key) {
        T* cache = static_cast<T*>(base) + (size_t)at.slot * a.ld;
        to = cache + (value ? a.kv_heads * a.kd + h * a.vd : h * a.kd);
    } else {
        to = static_cast<T*>(a.q) + (size_t)row * a.ldq + h * a.kd;
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int e = (c * 32 + l) * 4;
        if (e >= nd) break;
        float z[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
        if (w) {
            const float4 g = load4<VEC>(w, e, n);
            z[0] *= r * g.x;
            z[1] *= r * g.y;
            z[2] *= r * g.z;
            z[3] *= r * g.w;
        }
        if (e < rot) {
            if (!half) {
#pragma unroll
                for (int j = 0; j < 4; j += 2)
                    if (e + j < rot) {
                        const float co = cs[(e + j) / 2], si = sn[(e + j) / 2], p = z[j];
                        z[j] = fmaf(p, co, -(z[j + 1] * si));
                        z[j + 1] = fmaf(z[j + 1], co, p * si);
                    }
            } else {
                // the other half of the pairs comes from memory again (the lines are in L1) and is normed here too
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (e + j >= rot) break;
                    const bool first = e + j < hr;
                    const int i = first ? e + j : e + j - hr, o = first ? e + j + hr : i;
                    float p = x[o];
                    if (w) p *= r * w[o];
                    z[j] = first ? fmaf(z[j], cs[i], -(p * sn[i])) : fmaf(z[j], cs[i], p * sn[i]);
                }
            }
        }
        put4(to + e, make_float4(z[0], z[1], z[2], z[3]));
    }
}

template <class T, bool VEC>
static cudaError_t launch_qk(const QkArgs& a, dim3 grid, cudaStream_t q) {
    return std::max(a.kd, a.vd) <= 128 ? launch_pdl_try(k_fqk_rope<T, VEC, 1>, grid, dim3(QK_THREADS), 0, q, 1, a)
                                       : launch_pdl_try(k_fqk_rope<T, VEC, 2>, grid, dim3(QK_THREADS), 0, q, 1, a);
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
    const dim3 grid(gx, std::min(want, (a.n + (int)block.y - 1) / (int)block.y));
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
    if (op->seq.rows == 0 || op->seq.seqs == 0) return 0;
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
    a.lanes = 8;
    while (a.lanes < 32 && a.lanes * 4 < std::max(a.kd, a.vd)) a.lanes *= 2;
    const int per = QK_THREADS / a.lanes, units = a.heads + 2 * a.kv_heads;
    const dim3 grid(op->seq.rows, (units + per - 1) / per);
    const bool vec = aligned16(op->y) && op->ldy % 4 == 0 && op->q_off % 4 == 0 && op->k_off % 4 == 0 && op->v_off % 4 == 0 && op->dim % 4 == 0 &&
                     op->vdim % 4 == 0 && aligned16(op->q_norm) && aligned16(op->k_norm);
    cudaStream_t q = queue_of(st);
    cudaError_t e;
    if (op->dtype == DET_BF16) e = vec ? launch_qk<bf16, true>(a, grid, q) : launch_qk<bf16, false>(a, grid, q);
    else e = vec ? launch_qk<float, true>(a, grid, q) : launch_qk<float, false>(a, grid, q);
    return launched(name, e);
}

}  // extern "C"
