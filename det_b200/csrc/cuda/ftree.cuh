// Pieces shared by the ops of a step of drafted tokens (include/det_b200.h, det_tree_ref): refusals, which sequence a row belongs to,
// and how the attention's work is dealt out.
#pragma once
#include "fops.cuh"

namespace detb {

inline int refuse(const char* op, const char* why) {
    fprintf(stderr, "det_b200: %s refused: %s\n", op, why);
    return 1;
}
#define DETB_TAKE(cond, why)                   \
    do {                                       \
        if (!(cond)) return refuse(name, why); \
    } while (0)
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// The verdict of a launch as a return code.  A failed launch is no refusal: an earlier one of the same call may have been queued.
inline int launched(const char* op, cudaError_t e) {
    if (e == cudaSuccess) return 0;
    (void)cudaGetLastError();
    fprintf(stderr, "det_b200: %s: the launch failed: %s\n", op, cudaGetErrorString(e));
    return 1;
}
inline const char* bad_ref(const det_tree_ref& s) {
    if (s.seqs < 0 || s.rows < 0 || s.max_len < 0 || s.max_nodes < 0) return "negative sizes";
    if (s.seqs > 65535) return "too many sequences";
    if (s.seqs && s.rows && (!s.table || !s.first || !s.len)) return "table, first or len is NULL";
    return nullptr;
}

__device__ __forceinline__ void report_size(int* error_flag) { atomicExch(error_flag, DETB_ERR_SIZE); }

__device__ __forceinline__ void put4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void put4(bf16* p, float4 v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf(v.x, v.y), pack_bf(v.z, v.w)); }

// A cache pointer from device memory.
__device__ __forceinline__ bool usable_cache(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A sequence as device memory has it.  `bad`: its entries do not fit its cache (of `cap` rows) or the bounds of the call, and every op of the
// step leaves it out whole (it then has no rows here).  A sequence without rows has nothing that could not fit: a place that a batch leaves
// unused may hold anything.
struct TreeSpan {
    void* cache;
    int first, n, len;
    bool bad;
};
__device__ __forceinline__ TreeSpan tree_span(const det_tree_ref& s, int cap, int b) {
    TreeSpan t;
    const int next = s.first[b + 1];
    t.cache = s.table[b].cache;
    t.first = s.first[b];
    t.n = (int)((unsigned)next - (unsigned)t.first);           // no sum or difference of what was not checked before may overflow
    t.len = s.len[b];
    // (conditions joined without branches: k_fqk_rope has no registers to spare)
    t.bad = (t.n != 0) & ((t.first < 0) | (next < t.first) | (next > s.rows) | (t.n > s.max_nodes) | (t.n > cap) | (t.len < 0) |
                          (t.len > (int)((unsigned)cap - (unsigned)t.n)) | !usable_cache(t.cache));
    if (t.bad) t.n = 0;
    if (t.n == 0) t.len = 0;
    return t;
}
// The place of a row: its sequence's cache and the row there (negative: left out).  Called by whole warps with one row.
struct TreePlace {
    void* cache;
    int slot;
    bool nobodys;
};
__device__ __forceinline__ TreePlace tree_place(const det_tree_ref& s, int cap, int row, int lane) {
    int b = 0;
    for (int i = lane; i - lane < s.seqs; i += 32) b += __popc(__ballot_sync(FULL, i < s.seqs && s.first[i + 1] <= row));
    if (b >= s.seqs) return {nullptr, -1, true};
    const TreeSpan t = tree_span(s, cap, b);
    const unsigned node = (unsigned)row - (unsigned)t.first;
    return {t.cache, node < (unsigned)t.n ? t.len + (int)node : -1, false};
}

// ------------------------------------------------------------------------------------------------------ attention
// The query rows of a sequence and key/value head are (node, query head of the group) pairs, node first, in blocks of `block` rows;
// its keys come in tiles.  The tiles of all (sequence, row block, key/value head) segments, in that order, are dealt out evenly: CTA
// c takes `share` tiles from c * share on, whatever segments they belong to, so unequal lengths leave no CTA idle.  A segment that
// falls to one CTA is finished there; of the others every CTA leaves a piece (maximum, sum, values per row) in scratch, and the
// merge kernel adds the pieces in order of the keys.  A CTA has at most two such pieces, of its first and of its last stretch.  A CTA that
// passes from one segment to the next drains its pipeline in between: a segment counts for `turn` tiles more than it has, at its
// beginning, so that such CTAs get fewer.
constexpr int TREE_CTAS = 148;
constexpr int TREE_SHARE = 2;      // tiles of a CTA at least, if there are enough
constexpr int TREE_MAX_KEYS = 0x7fff0000;      // of a sequence: the end of its last tile fits 31 bits

struct TreeArgs {
    int heads, kv_heads, per_kv, dim, vdim, kd, vd, ld, ldq;
    unsigned long long per_magic;  // row / per_kv = row * per_magic >> 32, as row * per_kv < 2^32
    float scale2;                  // scale * log2(e)
    int cap;
    const void* q;
    const unsigned* mask;
    int mask_ld;
    const float* gate;
    int ldg;
    const int* pos;
    int rope_len;
    const float* vcs;
    const float* vsn;
    void* out;
    int ldo;
    float* part;                   // [CTA][2] pieces of tree_piece_floats(block, vd)
    void* maps;                    // [CTA][TREE_MAPS][2] tensor maps
    int* error_flag;
    int block, tile, blocks;       // rows of a block, keys of a tile, row blocks of the largest tree
    int ctas, turn;
    det_tree_ref seq;
};
constexpr int TREE_MAPS = 8;
constexpr size_t TREE_MAP_BYTES = (size_t)TREE_CTAS * TREE_MAPS * 2 * 128;
// A piece: {maximum, sum}[block] | values[block][vd].
__host__ __device__ constexpr size_t tree_piece_floats(int block, int vd) { return (size_t)block * (2 + vd); }

struct TreeSeg {
    int b, r0, rows;               // sequence, first row of the block, its rows
    int first, n, len, keys;       // first row of the step, nodes, cached rows, keys that some row of the block may see
    int edge;                      // keys that every row of the block sees
    int tiles;                     // 0: nothing to do (a sequence that does not fit is left out)
    bool bad;
};
__device__ __forceinline__ TreeSeg tree_seg(const TreeArgs& a, int seg) {
    TreeSeg s;
    s.b = seg / a.blocks;
    s.r0 = (seg - s.b * a.blocks) * a.block;
    const TreeSpan t = tree_span(a.seq, a.cap, s.b);
    s.first = t.first;
    s.n = t.n;
    s.len = t.len;
    s.bad = t.bad;
    s.rows = min(a.block, s.n * a.per_kv - s.r0);
    const int seen = a.mask ? s.n : min(s.n, (s.r0 + s.rows + a.per_kv - 1) / a.per_kv);
    s.keys = s.len + seen;
    s.edge = a.mask ? s.len : s.len + s.r0 / a.per_kv + 1;
    s.tiles = s.rows > 0 ? (s.keys + a.tile - 1) / a.tile : 0;
    return s;
}
// Places of a segment in the deal, for one key/value head: `turn`, then one for a tile, or two where it meets more than 128 rows (two
// slots of k_ftree_tc).  A tile goes to the CTA that has its last place.
__device__ __forceinline__ int tree_double(const TreeSeg& s) { return s.rows > 128 ? 1 : 0; }
__device__ __forceinline__ int tree_places(const TreeArgs& a, const TreeSeg& s) { return s.tiles > 0 ? (s.tiles << tree_double(s)) + a.turn : 0; }
__device__ __forceinline__ int tree_tiles(const TreeArgs& a, const TreeSeg& s, long long places) {      // of the segment's first places
    return (int)(max(0ll, places - a.turn) >> tree_double(s));
}
// Places of a CTA.
__device__ __forceinline__ long long tree_share(const TreeArgs& a, long long total) {
    if (total < 1ll << 31) return max(TREE_SHARE, (int)(((unsigned)total + a.ctas - 1) / (unsigned)a.ctas));
    return (total + a.ctas - 1) / a.ctas;
}
// Where a CTA's share begins and how long it is.  tree_start is called by a whole warp; every lane gets the result.
struct TreeShare {
    int seg, g, place;             // segment, key/value head, place within them
    long long left;                // places of the share
    int cta;                       // whose share it is
};
// With `segment` >= 0 it finds the share that begins first inside that segment (counted with the key/value heads) behind its first tile.
__device__ __forceinline__ TreeShare tree_start(const TreeArgs& a, int cta, int lane, long long* share_out = nullptr, int segment = -1) {
    const int segs = a.seq.seqs * a.blocks;
    long long total = 0;
    int mine = 0;                                             // places of the lane's last segment
    bool bad = false;
    for (int i = lane; i < segs; i += 32) {
        const TreeSeg s = tree_seg(a, i);
        total += mine = tree_places(a, s);
        bad |= s.bad;
    }
    if (cta == 0 && bad) report_size(a.error_flag);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(FULL, total, off);
    total *= a.kv_heads;
    const long long share = tree_share(a, total);
    if (share_out) *share_out = share;
    TreeShare w{0, 0, 0, 0, 0};
    if (segment >= 0) {
        w.seg = segment / a.kv_heads;
        w.g = segment - w.seg * a.kv_heads;
        long long before = 0;
        for (int i = lane; i < w.seg; i += 32) before += tree_places(a, tree_seg(a, i));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) before += __shfl_xor_sync(FULL, before, off);
        const TreeSeg s = tree_seg(a, w.seg);
        const int places = tree_places(a, s);
        const long long begin = before * a.kv_heads + (long long)w.g * places, first = begin + a.turn + tree_double(s);   // where its first tile goes
        if (places == 0) return w;
        w.cta = first + places < 1ll << 31 ? (int)((unsigned)first / (unsigned)share) : (int)(first / share);
        const long long border = (w.cta + 1) * share;
        w.place = (int)(border - begin);
        w.left = border < begin + places ? 1 : 0;
        return w;
    }
    const long long u0 = cta * share;
    if (u0 >= total) return w;
    if (segs <= 32 && total < 1ll << 31) {                     // the usual case in 32 bits
        int sum = mine * a.kv_heads;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(FULL, sum, off);
            if (lane >= off) sum += v;
        }
        const int src = __ffs(__ballot_sync(FULL, sum > (int)u0)) - 1, per = __shfl_sync(FULL, mine, src);
        const unsigned in = (unsigned)((int)u0 - __shfl_sync(FULL, sum - mine * a.kv_heads, src));
        return {src, (int)(in / (unsigned)per), (int)(in % (unsigned)per), min(share, total - u0), cta};
    }
    w.left = min(share, total - u0);
    w.cta = cta;
    long long base = 0;                                       // places ahead of these 32 segments
    for (int i = lane;; i += 32) {
        const int places = i >= segs ? 0 : segs <= 32 ? mine : tree_places(a, tree_seg(a, i));
        long long sum = (long long)places * a.kv_heads;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long v = __shfl_up_sync(FULL, sum, off);
            if (lane >= off) sum += v;
        }
        const unsigned holds = __ballot_sync(FULL, base + sum > u0);
        if (holds) {
            const int src = __ffs(holds) - 1, per = __shfl_sync(FULL, places, src);
            // places of the segment ahead of the share: below kv_heads * per, two for 64 keys of a head, 32 bytes each at least; more than
            // 32 bits of them would be a cache of 4 TB
            const unsigned in = (unsigned)(u0 - __shfl_sync(FULL, base + sum - (long long)places * a.kv_heads, src));
            w.seg = i - lane + src;
            w.g = (int)(in / (unsigned)per);
            w.place = (int)(in % (unsigned)per);
            return w;
        }
        base += __shfl_sync(FULL, sum, 31);
    }
}
// The next stretch of a share: `n` tiles from `tile` on of key/value head g of the segment; false when the share is done.
struct TreeItem {
    TreeSeg s;
    int g, tile, n;
    bool whole;                    // all tiles of the segment and head
    int piece;                     // else: which of the CTA's pieces
};
struct TreeWalk {
    TreeShare w;
    bool begun;
};
__device__ __forceinline__ bool tree_next(const TreeArgs& a, TreeWalk& k, TreeItem& it) {
    do {
        if (k.w.left <= 0) return false;
        it.s = tree_seg(a, k.w.seg);
        while (it.s.tiles == 0) {                              // only segments behind the first can be empty
            k.w.seg++;
            it.s = tree_seg(a, k.w.seg);
        }
        const int from = k.w.place, n = (int)min((long long)(tree_places(a, it.s) - from), k.w.left);
        it.g = k.w.g;
        it.tile = tree_tiles(a, it.s, from);
        it.n = tree_tiles(a, it.s, from + n) - it.tile;
        k.w.left -= n;
        k.w.place = 0;
        if (++k.w.g == a.kv_heads) {
            k.w.g = 0;
            k.w.seg++;
        }
    } while (it.n == 0);                                       // the share ended ahead of the first tile
    it.whole = it.n == it.s.tiles;
    it.piece = k.begun ? 1 : 0;
    k.begun = true;
    return true;
}
// Which of the 32 * W keys from c0 on a node sees, as bits; keys from the end of the tree on are never seen.  The words of the mask are
// asked for side by side.
template <int W>
__device__ __forceinline__ void tree_seen(const TreeArgs& a, const TreeSeg& s, int node, int c0, unsigned (&seen)[W]) {
    const int t0 = c0 - s.len, w0 = t0 >> 5, sh = t0 & 31;     // node of the first key (negative ahead of the tree), its word and bit
    unsigned m[W + 1];                                         // nodes 32 (w0 + i) ..
    const unsigned* row = a.mask ? a.mask + (size_t)(s.first + node) * a.mask_ld : nullptr;
    const int limit = a.mask ? s.n : min(s.n, node + 1);
#pragma unroll
    for (int i = 0; i <= W; i++) {
        const int n0 = (w0 + i) * 32, left = limit - n0;       // a word ahead of the tree is seen whole
        m[i] = n0 < 0 ? FULL : left <= 0 ? 0u : row ? row[w0 + i] : FULL;
        if (n0 >= 0 && left > 0 && left < 32) m[i] &= (1u << left) - 1u;
    }
#pragma unroll
    for (int i = 0; i < W; i++) seen[i] = __funnelshift_r(m[i], m[i + 1], sh);
}
// A finished head of a row: elements v .. v + 3 are turned back, gated and stored.
template <class T>
struct TreeOut {
    T* out;
    const float* c;                // turn of the row's position, or NULL
    const float* s;
    float w;
    int vdim;
    bool skip;
    __device__ __forceinline__ TreeOut(const TreeArgs& a, int row, int h)
        : out(static_cast<T*>(a.out) + (size_t)row * a.ldo + (size_t)h * a.vdim), c(nullptr), s(nullptr), w(1.0f), vdim(a.vdim), skip(false) {
        if (a.vcs) {
            const int pos = a.pos[row];
            skip = pos < 0 || pos >= a.rope_len;
            if (skip) report_size(a.error_flag);
            c = a.vcs + (size_t)(skip ? 0 : pos) * (a.vdim / 2);
            s = a.vsn + (size_t)(skip ? 0 : pos) * (a.vdim / 2);
        }
        if (a.gate) w = sigmoid_fast(a.gate[(size_t)row * a.ldg + h]);
    }
    // ... turned back and gated
    __device__ __forceinline__ float4 finished(int v, float4 x) const {
        float o[4] = {x.x * w, x.y * w, x.z * w, x.w * w};
        if (c) {
#pragma unroll
            for (int j = 0; j < 4; j += 2)
                if (v + j < vdim) {
                    const float cj = c[(v + j) / 2], sj = s[(v + j) / 2], u = o[j];
                    o[j] = fmaf(u, cj, o[j + 1] * sj);
                    o[j + 1] = fmaf(o[j + 1], cj, -(u * sj));
                }
        }
        return make_float4(o[0], o[1], o[2], o[3]);
    }
    __device__ __forceinline__ void put4at(int v, float4 x) const {
        if (skip) return;
        x = finished(v, x);
        const float o[4] = {x.x, x.y, x.z, x.w};
        T* to = out + v;
        if (v + 4 <= vdim && (reinterpret_cast<uintptr_t>(to) & (4 * sizeof(T) - 1)) == 0) {
            put4(to, x);
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (v + j < vdim) put(to + j, o[j]);
    }
};
__device__ __forceinline__ float4 scaled4(float4 v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }

__device__ __forceinline__ void add4(float4& o, float f, float4 x) {
    o.x = fmaf(f, x.x, o.x);
    o.y = fmaf(f, x.y, o.y);
    o.z = fmaf(f, x.z, o.z);
    o.w = fmaf(f, x.w, o.w);
}

// Lets the kernel have the dynamic shared memory of its largest call.  Every call sets the same limit, since calls of other sizes may run
// on other threads; 1 KB is left for what the kernels declare themselves.
constexpr int TREE_SMEM = 226 * 1024;
template <class F>
inline cudaError_t most_smem(F* kernel) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TREE_SMEM); }

// ftree_few.cu: bfloat16 activations, few rows.
bool ftree_few_takes(const TreeArgs& a, int rows);
void ftree_few_shape(int* block, int* tile);
cudaError_t ftree_few_launch(const TreeArgs& a, cudaStream_t q);
// ftree_tc.cu: bfloat16 activations.  Rows of a block, keys of a tile and the tiles that a turn costs are the kernel's.
void ftree_tc_shape(int rows, int kd, int vd, int* block, int* tile, int* turn);
cudaError_t ftree_tc_launch(const TreeArgs& a, cudaStream_t q);

}  // namespace detb
