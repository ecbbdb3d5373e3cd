// Tree attention over bfloat16 caches on the tensor cores: tcgen05.mma kind::f16, scores and outputs in TMEM, one pass over the keys.
//
// A slot is 128 query rows (TMEM lanes) with scores S = Q K^T [128 x keys of a tile], weights P over the same columns (bfloat16, read
// by the second product straight from TMEM) and outputs O += P V [128 x vd].  A thread of a slot's four warps owns one row: running
// reference, sum and weights of its scores need no exchange.  The reference moves (and O is scaled) only when a row's maximum has
// grown by more than 2^8 over it, so the weights stay below 2^8 and O is touched rarely.
//
// Two slots per CTA take turns, so that the products of one run beside the exponentials of the other.  Up to 128 rows: both hold the
// same rows and take every other tile of keys, and their results are added at the end; more rows: 128 rows each over the same tiles.
// Heads above 128: one slot, tiles of 64 keys, and products and softmax take turns, which costs them (512 rows behind 4096, 16 / 2 heads of
// 256: 75 us, 487 TFLOP/s).  It is not what TMEM and shared memory could hold: heads of 192 with values of 128 would have room for two
// slots, heads of 256 for a second set of scores.
//
// Warps: four per slot for the softmax; one that loads tiles of K and V (TMA, 128-byte swizzle; K K-major, V as it lies in the cache,
// MN-major); one that issues the products; two that bring the query rows (16-byte asynchronous copies, a head's rows are not evenly
// spaced) and look through the values of tiles that not every row sees.  The caches' addresses and lengths are in device memory: the
// loading warp writes them into a tensor map of its CTA (tensormap.replace) when a stretch begins another sequence, and rows behind the
// last key then read as zeros.
//
// A masked weight is zero, but zero times a value that is not finite is not: in tiles that not every row sees such values enter the
// product as zeros, and the end of the stretch adds them to the rows that do see them.
//
// A weight is rounded to bfloat16 for its product, as any tensor-core form must (half a step, 2^-8 relative, independent from key to
// key); sums and references are fp32.
//
// What bounds it (40 / 8 heads of 128).  Trees of 16 nodes read the cache once: 16 nodes behind 65536 keys 63 us (269 MB from HBM, what
// they cannot do without), 32 sequences of 16 behind 4096 keys 104 us (5.2 TB/s).  A prompt of 2048 behind 6144 takes 332 us with inputs
// that change from call to call (905 TFLOP/s) and 300 to 306 with inputs that stay (984 to 1001), 20 of them the merge: a tile of 128 rows x
// 128 keys is 1040 cycles of products (measured alone), beside the tiles' copies into the same shared memory; then comes the chain from scores
// over a warp's exponentials (about 1600 cycles) to the weights, which two slots hide in part.  The pipe is busy 52 % of the attention
// kernel's time there, 41 % with 512 rows, 40 % with a tree of 61 behind 32749 (80 to 84 us).  The softmax of a slot has 168 registers a
// thread, with spills, and waits for each load of TMEM before it asks for the next.  The products are issued by an elected lane: by a branch
// on the lane's number, operands went through vector registers and the issue was the bound (358 us).  Measured with inputs that stay, and not
// taken: copies of the tiles by warps in place of TMA (prompt 532 us against 401), tiles of 64 keys with two score buffers (515 against 354), a
// product warp for each slot (405 against 354), TMEM loads of 16 columns asked for ahead (369 against 354), a polynomial in place of an
// eighth to three eighths of the ex2 (312 to 331 against 306).
#include "ftree.cuh"
#include "umma.cuh"
#include <algorithm>

namespace detb {

constexpr int TT_ROWS = 128;
constexpr int TT_COPY = 64;                          // threads that bring rows
constexpr float TT_GROWTH = 8.0f;                   // log2 of how far a maximum may outgrow the reference

template <int SLOTS, int KT>
struct TtCfg {
    static constexpr int SOFT = 4 * SLOTS, LOADS = SOFT, PRODUCTS = SOFT + 1, ROWS = SOFT + 2, THREADS = (SOFT + 4) * 32;   // first warps of the roles
    static constexpr int O_COL = SLOTS * KT;
};
struct TtShape {
    int nkb, nvb;                                   // 64-element blocks of a key, of a value
    int stages, stage_bytes;
    int twice;                                      // blocks of 128 rows: one slot's room holds the next stretch's rows
    int q_bytes;                                    // of one slot's rows
};

constexpr int TT_STAGES = 12;
struct alignas(128) TtTables {
    unsigned char map[2][128];
    unsigned long long raw[TT_STAGES];               // a tile of values that is looked through before it is full
    unsigned long long full[TT_STAGES], empty[TT_STAGES], q_full[2], q_empty[2], s_full[2], p_full[2], o_full, o_empty;
    float2 ml[2][TT_ROWS];                           // [slot]: reference and sum of a row
    TreeShare share;
    unsigned tmem_slot;
    int odd[4];                                      // number (+ 1) of the stretch whose values were not all finite
};

__device__ __forceinline__ void umma_f16_ss(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(unsigned d, unsigned a, unsigned long long b, unsigned idesc, unsigned acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// MN-major, SWIZZLE_128B: 64 neighbouring values of a key per 128-byte row, 8-key groups 1024 bytes apart, blocks of 64 values `lead`
// bytes apart.
__device__ __forceinline__ unsigned long long umma_desc_mn(const void* smem, unsigned lead) {
    const unsigned addr = smem_addr(smem);
    unsigned long long d = 0;
    d |= (unsigned long long)((addr & 0x3FFFF) >> 4);
    d |= (unsigned long long)(lead >> 4) << 16;
    d |= (unsigned long long)(1024 >> 4) << 32;
    d |= (unsigned long long)1 << 46;
    d |= (unsigned long long)2 << 61;
    return d;
}
// fp32 accumulator, bfloat16 operands, M = 128, N = n; b_mn: B is MN-major.
__device__ __forceinline__ unsigned tt_idesc(int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((unsigned)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tmem_st(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {      // relative error about 2^-22; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two neighbouring fp32 values in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)), "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
// Waits for the loads of TMEM; what they brought is not used before.
__device__ __forceinline__ void tmem_landed(int (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                   "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                   "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_landed(int (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void copy16(unsigned dst, const void* src, int bytes) {      // what is missing of 16 bytes becomes zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// One lane of the warp, which the compiler then knows to be alone: operands of tcgen05.mma and TMA stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
    unsigned x;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
    return x != 0;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The tensor maps of a sequence's keys and values, made from the launch's by the whole warp: their addresses and number of rows are set
// in shared memory and the maps copied to `to`, where loads may name them.
__device__ __forceinline__ void tt_maps(const CUtensorMap& mk, const CUtensorMap& mv, unsigned char (*sm)[128], const bf16* keys, const bf16* values, int rows,
                                        unsigned char* to, int lane) {
    reinterpret_cast<unsigned*>(sm[0])[lane] = reinterpret_cast<const unsigned*>(&mk)[lane];
    reinterpret_cast<unsigned*>(sm[1])[lane] = reinterpret_cast<const unsigned*>(&mv)[lane];
    __syncwarp();
    if (lane < 2) {
        const unsigned m = smem_addr(sm[lane]);
        asm volatile("tensormap.replace.tile.global_address.shared::cta.b1024.b64 [%0], %1;" ::"r"(m), "l"(lane ? values : keys) : "memory");
        asm volatile("tensormap.replace.tile.global_dim.shared::cta.b1024.b32 [%0], 2, %1;" ::"r"(m), "r"(rows) : "memory");
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; i++) reinterpret_cast<unsigned*>(to + i * 128)[lane] = reinterpret_cast<const unsigned*>(sm[i])[lane];
    __syncwarp();
    if (lane == 0) {                                 // the lane that names them: one release for both
        asm volatile("fence.proxy.tensormap::generic.release.gpu;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 2; i++) asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(to + i * 128) : "memory");
    }
}
__device__ __forceinline__ void tt_load(void* dst, const void* map, int x, int head, int row, unsigned long long* bar, unsigned long long policy) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(
                     smem_addr(dst)),
                 "l"(map), "r"(x), "r"(head), "r"(row), "r"(smem_addr(bar)), "l"(policy)
                 : "memory");
}
// Values that are not finite become zeros in the keys r0 .. r1 of a staged tile (blocks of 64 columns, 128 bytes a key); true when there
// were any.
template <int KT>
__device__ __forceinline__ bool tt_clean(uint8_t* tile, int blocks, int r0, int r1, int tid) {
    bool odd = false;
    for (int b = 0; b < blocks; b++)
#pragma unroll 4
        for (int i = r0 * 128 + tid * 16; i < r1 * 128; i += TT_COPY * 16) {
            uint4* p = reinterpret_cast<uint4*>(tile + b * KT * 128 + i);
            const uint4 v = *p;
            // an exponent of ones carries into the sign's place
            auto carry = [](unsigned w) { return (w & 0x7f807f80u) + 0x00800080u; };
            if (!((carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & 0x80008000u)) continue;
            unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if ((w[j] & 0x7f80u) == 0x7f80u) w[j] &= 0xffff0000u;
                if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] &= 0xffffu;
            }
            *p = make_uint4(w[0], w[1], w[2], w[3]);
            odd = true;
        }
    return odd;
}

// The largest of a row's scores in the KT columns from `ts` on; MASKED: of those it sees.
template <int KT, bool MASKED>
__device__ __forceinline__ float tt_max(unsigned ts, const unsigned (&words)[KT / 32]) {
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
    for (int q = 0; q < KT / 32; q++) {
        int v[32];
        tmem_ld(ts + q * 32, v);
        unsigned seen = FULL;
        if (MASKED) {
#pragma unroll
            for (int i = 0; i < KT / 32; i++) seen = i == q ? words[i] : seen;
        }
        tmem_landed(v);
#pragma unroll
        for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], !MASKED || (seen >> i) & 1u ? __int_as_float(v[i]) : -INFINITY);
    }
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// Weights of scores that are not masked in one pass: 2^(score * scale + base) into w, bfloat16 pairs, and their sum; returns the largest
// score.
template <int KT>
__device__ __forceinline__ float tt_one_pass(unsigned ts, float scale2, float base, unsigned (&w)[KT / 2], float& total) {
    const float2 scale = make_float2(scale2, scale2), off = make_float2(base, base);
    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int q = 0; q < KT / 32; q++) {
        int v[32];
        tmem_ld(ts + q * 32, v);
        tmem_landed(v);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float a = __int_as_float(v[i]), b = __int_as_float(v[i + 1]);
            asm("max.f32 %0, %0, %1, %2;" : "+f"(top[(i >> 1) & 1]) : "f"(a), "f"(b));
            const float2 x = fma2(make_float2(a, b), scale, off);
            const float2 p = make_float2(ex2(x.x), ex2(x.y));
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], p);
            w[q * 16 + i / 2] = pack_bf(p.x, p.y);
        }
    }
    total = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    return fmaxf(top[0], top[1]);
}
// The row's weights 2^(score * scale + base) in place of its scores; returns their sum.
template <int KT, bool MASKED>
__device__ __forceinline__ float tt_weights(unsigned ts, const unsigned (&words)[KT / 32], float scale2, float base) {
    const float2 scale = make_float2(scale2, scale2), off = make_float2(base, base);
    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll 1
    for (int q = 0; q < KT / 32; q++) {
        int v[32];
        tmem_ld(ts + q * 32, v);
        unsigned seen = FULL;
        if (MASKED) {
#pragma unroll
            for (int i = 0; i < KT / 32; i++) seen = i == q ? words[i] : seen;
        }
        tmem_landed(v);
        unsigned w[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 x = fma2(make_float2(__int_as_float(v[i]), __int_as_float(v[i + 1])), scale, off);
            float2 p = make_float2(ex2(x.x), ex2(x.y));
            if (MASKED) p = make_float2((seen >> i) & 1u ? p.x : 0.0f, (seen >> (i + 1)) & 1u ? p.y : 0.0f);
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], p);
            w[i / 2] = pack_bf(p.x, p.y);
        }
        tmem_st(ts + q * 16, w);
    }
    return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

// Eight lanes exchange: lane l had piece k of its row in x[k], afterwards it has piece l of row k (N words each).
template <int N>
__device__ __forceinline__ void tt_turn(unsigned (&x)[8][N], int lane) {
#pragma unroll
    for (int s = 1; s < 8; s *= 2) {
        const bool up = lane & s;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (k & s) continue;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const unsigned y = __shfl_xor_sync(FULL, up ? x[k][i] : x[k + s][i], s);
                if (up) x[k][i] = y;
                else x[k + s][i] = y;
            }
        }
    }
}

template <int SLOTS, int KT>
__global__ void __launch_bounds__(TtCfg<SLOTS, KT>::THREADS, 1) k_ftree_tc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                               const TreeArgs a, const TtShape sh) {
    using Cfg = TtCfg<SLOTS, KT>;
    constexpr int SOFT = Cfg::SOFT, LOADS = Cfg::LOADS, PRODUCTS = Cfg::PRODUCTS, ROWS = Cfg::ROWS;
    extern __shared__ __align__(1024) uint8_t Qs[];                     // [SLOTS][nkb][128][128 B], the ring, the tables
    uint8_t* ring = Qs + SLOTS * sh.q_bytes;
    TtTables& tb = *reinterpret_cast<TtTables*>(ring + (size_t)sh.stages * sh.stage_bytes);
    auto &full = tb.full, &empty = tb.empty, &raw = tb.raw;
    auto &q_full = tb.q_full, &q_empty = tb.q_empty, &s_full = tb.s_full, &p_full = tb.p_full;
    auto &o_full = tb.o_full, &o_empty = tb.o_empty;
    auto &odd = tb.odd;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long wl = wait_limit(a.error_flag);
    if (smem_addr(Qs) & 1023) {                      // the layout of the operands needs it
        pdl_wait();
        pdl_trigger();
        if (threadIdx.x == 0) report_size(a.error_flag);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < sh.stages; s++) {
            mbar_init(&raw[s], 1);
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 2);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        mbar_init(&o_full, 1);
        mbar_init(&o_empty, SOFT);
        for (int i = 0; i < 4; i++) odd[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == PRODUCTS) tmem_alloc(&tb.tmem_slot, 512);
    pdl_wait();
    pdl_trigger();                                   // behind the wait: what k_ftree_merge reads ahead of its own is then there
    if (warp == 0) {
        const TreeShare w = tree_start(a, blockIdx.x, lane);
        if (lane == 0) tb.share = w;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tb.tmem_slot;
    TreeWalk walk{tb.share, false};
    TreeItem it;
    bool ok = true;
    auto wait = [&](unsigned long long* bar, unsigned parity) { return __all_sync(FULL, mbar_wait(bar, parity, wl)) != 0; };   // by whole warps
    const bool twice = sh.twice != 0;
    // the slots take every other tile of the same rows; tiles whose scores are asked for ahead
    auto both_of = [](const TreeItem& x) { return SLOTS == 2 && x.s.rows <= TT_ROWS; };
    auto lead_of = [&](const TreeItem& x) { return both_of(x) ? 2 : 1; };
    unsigned item = 0;                               // stretches so far

    if (warp == LOADS) {
        // ---- tiles of keys and values
        unsigned c = 0, sn = 0, phase = 0;           // tiles issued, place in the ring
        int seq = -1, maps = 0;
        unsigned char* map = nullptr;
        // keys that one row block reads are read once: they leave the L2 cache to the pieces and to the next kernels
        unsigned long long policy;
        if (a.blocks == 1) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
        while (ok && tree_next(a, walk, it)) {
            const TreeSeg& s = it.s;
            if (s.b != seq) {
                // a map is written again TREE_MAPS sequences later: by then more tiles have passed the ring than it has stages
                const bf16* cache = static_cast<const bf16*>(a.seq.table[s.b].cache);
                map = static_cast<unsigned char*>(a.maps) + ((size_t)blockIdx.x * TREE_MAPS + maps % TREE_MAPS) * 256;
                tt_maps(map_k, map_v, tb.map, cache, cache + a.kv_heads * a.kd, s.len + s.n, map, lane);
                seq = s.b;
                maps++;
            }
            const int lead = lead_of(it);
            if (lane == 0) {
                auto fetch = [&](bool value, int t) {
                    if (c >= (unsigned)sh.stages) ok = mbar_wait(&empty[sn], phase ^ 1u, wl);
                    if (!ok) return;
                    const int k0 = (it.tile + t) * KT, blocks = value ? sh.nvb : sh.nkb;
                    const bool look = value && k0 + KT > s.edge;
                    unsigned long long* bar = look ? &raw[sn] : &full[sn];
                    mbar_expect_tx(bar, blocks * KT * 128);
                    if (!look) mbar_arrive(bar);
                    for (int i = 0; i < blocks; i++)
                        tt_load(ring + (size_t)sn * sh.stage_bytes + i * KT * 128, map + (value ? 128 : 0), i * 64, it.g, k0, bar, policy);
                    c++;
                    if (++sn == (unsigned)sh.stages) sn = 0, phase ^= 1u;
                };
                for (int t = 0; t < min(lead, it.n) && ok; t++) fetch(false, t);
                for (int t = 0; t < it.n && ok; t++) {
                    fetch(true, t);
                    if (ok && t + lead < it.n) fetch(false, t + lead);
                }
            }
            ok = __shfl_sync(FULL, ok ? 1 : 0, 0) != 0;
        }
        if (!ok && lane == 0)                        // the loads in flight write shared memory: at the most one phase of each barrier is open
            for (unsigned k = 1; k <= (unsigned)sh.stages && k <= c; k++) {
                (void)mbar_wait(&full[(c - k) % sh.stages], ((c - k) / sh.stages) & 1u, wl);
            }
    } else if (warp >= ROWS) {
        // ---- query rows, and values that not every row sees
        const int tid = threadIdx.x - ROWS * 32;
        const int kp = (a.kd + 15) / 16 * 2, lanes = kp <= 8 ? 8 : kp <= 16 ? 16 : 32, qc = lane % lanes, qstep = TT_COPY / lanes;
        const int head_step = qstep % a.per_kv;      // from a thread's row to its next one: heads, and elements without and with one more node
        const ptrdiff_t ahead = (ptrdiff_t)(qstep / a.per_kv) * a.ldq + head_step * a.kd, wrap = (ptrdiff_t)a.ldq - a.per_kv * a.kd;
        unsigned c = 0, looked = 0;                  // tiles of the stretches before; phases of `raw`, a bit per stage
        while (ok && tree_next(a, walk, it)) {
            const TreeSeg& s = it.s;
            const int qb = twice ? item & 1 : 0, lead = lead_of(it);
            if (item >= (twice ? 2u : 1u)) ok = wait(&q_empty[qb], ((twice ? item >> 1 : item) & 1u) ^ 1u);
            if (!ok) break;
            // a row per `lanes` lanes; rows that are not there keep what is there (a row's scores are its own)
            const bf16* q = static_cast<const bf16*>(a.q) + (size_t)s.first * a.ldq + (size_t)it.g * a.per_kv * a.kd;
            if (qc < kp) {
                const int row = s.r0 + tid / lanes, node = (int)(row * a.per_magic >> 32);
                int head = row - node * a.per_kv;
                const bf16* src = q + (size_t)node * a.ldq + head * a.kd + (qc * 8 < a.kd ? qc * 8 : 0);
                const int bytes = qc * 8 < a.kd ? 16 : 0;
                const unsigned dst = smem_addr(Qs) + (unsigned)((twice ? qb * sh.q_bytes : 0) + (qc >> 3) * TT_ROWS * 128);
#pragma unroll 4
                for (int r = tid / lanes; r < s.rows; r += qstep) {
                    const unsigned half = r >= TT_ROWS ? (unsigned)(sh.q_bytes - TT_ROWS * 128) : 0u;       // the second slot's rows
                    copy16(dst + half + (unsigned)(r * 128 + (((qc ^ r) & 7) << 4)), src, bytes);
                    src += ahead;
                    head += head_step;
                    if (head >= a.per_kv) {
                        head -= a.per_kv;
                        src += wrap;
                    }
                }
            }
            copies_wait_all();
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[qb]);
            for (int t = max(0, s.edge / KT - it.tile); t < it.n && ok; t++) {
                // the ring holds K .. (lead tiles), then V, K, V, K ..
                const unsigned at = c + min(lead, it.n) + t + min(t, max(0, it.n - lead)), sn = at % sh.stages;
                ok = wait(&raw[sn], (looked >> sn) & 1u);
                looked ^= 1u << sn;
                if (!ok) break;
                const int k0 = (it.tile + t) * KT;
                if (tt_clean<KT>(ring + (size_t)sn * sh.stage_bytes, sh.nvb, max(0, s.edge - k0), min(KT, s.len + s.n - k0), tid))
                    *reinterpret_cast<volatile int*>(&odd[item & 3]) = (int)item + 1;
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[sn]);
            }
            c += 2 * it.n;
            item++;
        }
    } else if (warp == PRODUCTS) {
        // ---- products
        if (elect_one()) {
            const unsigned id_s = tt_idesc(KT, false), vn = (unsigned)(a.vd + 15) / 16 * 16, id_o = tt_idesc((int)vn, true);
            const int ksteps = (a.kd + 15) / 16;
            const unsigned long long q_desc = umma_desc(Qs), k_desc = umma_desc(ring), v_desc = umma_desc_mn(ring, KT * 128);
            unsigned c = 0, phase = 0, np[2] = {0, 0};   // place in the ring, weights taken per slot
            while (ok && tree_next(a, walk, it)) {
                const int qb = twice ? item & 1 : 0, lead = lead_of(it);
                const bool both = both_of(it), second = it.s.rows > TT_ROWS;
                ok = mbar_wait(&q_full[qb], ((twice ? item >> 1 : item) & 1u), wl);
                if (!ok) break;
                // descriptors of neighbouring steps differ in their address (units of 16 bytes) only
                auto scores = [&](int slot, unsigned s) {
                    unsigned long long q = q_desc + (unsigned)(twice ? qb : both ? 0 : slot) * (unsigned)(sh.q_bytes >> 4), k = k_desc + s * (unsigned)(sh.stage_bytes >> 4);
                    for (int e = 0; e < ksteps; e += 4) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (e + i < ksteps) umma_f16_ss(tmem + slot * KT, q + 2 * i, k + 2 * i, id_s, (e | i) ? 1u : 0u);
                        q += TT_ROWS * 128 >> 4;
                        k += KT * 128 >> 4;
                    }
                    umma_commit(&s_full[slot]);
                };
                auto outputs = [&](int slot, unsigned s, bool first) {
                    const unsigned long long v = v_desc + s * (unsigned)(sh.stage_bytes >> 4);
#pragma unroll
                    for (int k = 0; k < KT / 16; k++)
                        umma_f16_ts(tmem + Cfg::O_COL + slot * (256 / SLOTS), tmem + slot * KT + k * 8, v + k * 128, id_o, first && k == 0 ? 0u : 1u);
                };
                auto stage = [&]() {
                    const unsigned s = c;
                    ok = mbar_wait(&full[s], phase, wl);
                    if (++c == (unsigned)sh.stages) c = 0, phase ^= 1u;
                    tc_fence_after();
                    return s;
                };
                auto weights = [&](int slot) {
                    ok = mbar_wait(&p_full[slot], np[slot] & 1u, wl);
                    np[slot]++;
                    tc_fence_after();
                };
                for (int t = 0; t < min(lead, it.n) && ok; t++) {
                    const unsigned s = stage();
                    if (!ok) break;
                    scores(both ? t & 1 : 0, s);
                    if (second) scores(1, s);
                    umma_commit(&empty[s]);
                    if (t + 1 == it.n) umma_commit(&q_empty[qb]);
                }
                for (int t = 0; t < it.n && ok; t++) {
                    const unsigned sv = stage();
                    if (!ok) break;
                    if (t == 0 && item > 0) {        // the outputs of the stretch before have been read
                        ok = mbar_wait(&o_empty, (item & 1u) ^ 1u, wl);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    const int slot = both ? t & 1 : 0;
                    const bool more = t + lead < it.n;
                    unsigned sk = 0;
                    weights(slot);
                    if (!ok) break;
                    outputs(slot, sv, both ? t < 2 : t == 0);
                    if (!second) umma_commit(&empty[sv]);
                    if (more) {
                        sk = stage();
                        if (!ok) break;
                        scores(slot, sk);
                    }
                    if (second) {
                        weights(1);
                        if (!ok) break;
                        outputs(1, sv, t == 0);
                        umma_commit(&empty[sv]);
                        if (more) scores(1, sk);
                    }
                    if (more) {
                        umma_commit(&empty[sk]);
                        if (t + lead + 1 == it.n) umma_commit(&q_empty[qb]);
                    }
                }
                if (ok) umma_commit(&o_full);
                item++;
            }
        }
        ok = __all_sync(FULL, ok) != 0;
    } else {
        // ---- softmax
        const int slot = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const unsigned lanes = (unsigned)(quarter * 32) << 16;
        const unsigned ts = tmem + lanes + slot * KT, to = tmem + lanes + Cfg::O_COL + slot * (256 / SLOTS);
        unsigned ns = 0;                             // scores taken
        // after an expired wait the stretches are gone through without waiting, so that all warps meet at the barrier below
        while (tree_next(a, walk, it)) {
            const TreeSeg& s = it.s;
            const bool both = both_of(it);
            const int br = both ? r : slot * TT_ROWS + r;                     // row of the block
            const bool mine = br < s.rows, any = (both ? quarter * 32 : slot * TT_ROWS + quarter * 32) < s.rows;
            const int row = s.r0 + min(br, s.rows - 1), node = row / a.per_kv;
            float m = -INFINITY, l = 0.0f;
            const int jobs = both ? (it.n + 1 - slot) / 2 : it.n;
            for (int j = 0; j < jobs; j++) {
                const int k0 = (it.tile + (both ? 2 * j + slot : j)) * KT;
                const bool tree = k0 + KT > s.edge;
                unsigned seen[KT / 32];
                if (tree && any) tree_seen<KT / 32>(a, s, node, k0, seen);
                if (ok) ok = wait(&s_full[slot], ns & 1u);
                ns++;
                tc_fence_after();
                if (any) {
                    // as a rule the reference holds: weights in one pass, stored when the tile's maximum is known not to have outgrown it
                    float mt;
                    bool done = false;
                    if (!tree && j > 0) {
                        unsigned w[KT / 2];
                        float sum;
                        mt = tt_one_pass<KT>(ts, a.scale2, m == -INFINITY ? 0.0f : -m * a.scale2, w, sum);
                        done = !__any_sync(FULL, (mt - m) * a.scale2 > TT_GROWTH);
                        if (done) {
                            l += sum;
#pragma unroll
                            for (int q = 0; q < KT / 32; q++) {
                                unsigned x[16];
#pragma unroll
                                for (int i = 0; i < 16; i++) x[i] = w[q * 16 + i];
                                tmem_st(ts + q * 16, x);
                            }
                        }
                    } else {
                        mt = tree ? tt_max<KT, true>(ts, seen) : tt_max<KT, false>(ts, seen);
                    }
                    if (!done) {
                        const bool grow = (mt - m) * a.scale2 > TT_GROWTH;
                        if (__any_sync(FULL, grow)) {
                            const float f = grow ? ex2((m - mt) * a.scale2) : 1.0f;
                            if (grow) m = mt;
                            l *= f;
                            __syncwarp();
                            if (j > 0) {
#pragma unroll 1
                                for (int q = 0; q < a.vd; q += 16) {
                                    int v[16];
                                    tmem_ld(to + q, v);
                                    tmem_landed(v);
                                    unsigned w[16];
#pragma unroll
                                    for (int i = 0; i < 16; i++) w[i] = __float_as_uint(__int_as_float(v[i]) * f);
                                    tmem_st(to + q, w);
                                }
                            }
                        }
                        const float base = m == -INFINITY ? 0.0f : -m * a.scale2;
                        l += tree ? tt_weights<KT, true>(ts, seen, a.scale2, base) : tt_weights<KT, false>(ts, seen, a.scale2, base);
                    }
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[slot]);
            }
            if (ok) ok = wait(&o_full, item & 1u);
            tc_fence_after();
            // ---- end of the stretch
            float f0 = 1.0f, f1 = 0.0f;
            bool other = false;
            if (both) {
                asm volatile("bar.sync 1, %0;" ::"n"(SOFT * 32) : "memory");   // the last stretch's have been read
                tb.ml[slot][r] = make_float2(m, l);
                asm volatile("bar.sync 1, %0;" ::"n"(SOFT * 32) : "memory");
                other = it.n > 1;                     // else the second slot had no tile and its outputs hold nothing
                const float2 x = tb.ml[0][r], y = tb.ml[1][r];
                m = fmaxf(x.x, y.x);
                const float b = m == -INFINITY ? 0.0f : m;
                f0 = ex2((x.x - b) * a.scale2);
                f1 = ex2((y.x - b) * a.scale2);
                l = f0 * x.y + f1 * y.y;
            }
            if (any) {
                const unsigned o0 = tmem + lanes + Cfg::O_COL + (both ? 0 : slot * (256 / SLOTS)), o1 = o0 + 256 / SLOTS;
                const bool fix = *reinterpret_cast<volatile int*>(&odd[item & 3]) == (int)item + 1;
                const int orow = s.first + node, h = it.g * a.per_kv + row % a.per_kv;
                const TreeOut<bf16> out(a, orow, h);
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                float* piece = a.part + ((size_t)blockIdx.x * 2 + it.piece) * tree_piece_floats(a.block, a.vd);
#pragma unroll 1
                for (int q = both ? slot * 32 : 0; q < a.vd; q += both ? 64 : 32) {
                    int v[32], w[32];
                    tmem_ld(o0 + q, v);
                    if (other) tmem_ld(o1 + q, w);
                    tmem_landed(v);
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = __int_as_float(v[i]) * f0;
                    if (other) {
                        tmem_landed(w);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = fmaf(__int_as_float(w[i]), f1, o[i]);
                    }
                    if (fix) {                        // warps agree on it
                        // values of attended nodes that are not finite (they entered the product as zeros)
                        const int k1 = min(s.len + s.n, (it.tile + it.n) * KT);
#pragma unroll 1
                        for (int k = max(it.tile * KT, s.edge); k < k1; k++) {
                            unsigned sees[1];
                            tree_seen<1>(a, s, node, k, sees);
                            if (!(sees[0] & 1u)) continue;
                            const bf16* val = static_cast<const bf16*>(a.seq.table[s.b].cache) + (size_t)k * a.ld + a.kv_heads * a.kd + it.g * a.vd + q;
#pragma unroll
                            for (int i = 0; i < 32; i++) {
                                const float x = q + i < a.vd ? to_f(val[i]) : 0.0f;
                                if (!isfinite(x)) o[i] += x;
                            }
                        }
                    }
                    // eight lanes store a row's 32 values side by side, row after row (a lane per row would touch 32 lines at a time)
                    const int group = lane & 24, col = q + (lane & 7) * 4;
                    if (it.whole) {
                        unsigned x[8][2];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float4 y = out.finished(q + i * 4, make_float4(o[i * 4] * inv, o[i * 4 + 1] * inv, o[i * 4 + 2] * inv, o[i * 4 + 3] * inv));
                            x[i][0] = pack_bf(y.x, y.y);
                            x[i][1] = pack_bf(y.z, y.w);
                        }
                        tt_turn<2>(x, lane);
                        const unsigned long long own = mine && !out.skip ? reinterpret_cast<unsigned long long>(out.out) : 0;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            bf16* to = reinterpret_cast<bf16*>(__shfl_sync(FULL, own, group + k));
                            if (!to || col >= a.vdim) continue;
                            to += col;
                            if (col + 4 <= a.vdim && (reinterpret_cast<uintptr_t>(to) & 7) == 0) {
                                *reinterpret_cast<uint2*>(to) = make_uint2(x[k][0], x[k][1]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++)
                                    if (col + j < a.vdim) reinterpret_cast<unsigned short*>(to)[j] = (unsigned short)(x[k][j >> 1] >> (j & 1) * 16);
                            }
                        }
                    } else {
                        unsigned x[8][4];
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i >> 2][i & 3] = __float_as_uint(o[i]);
                        tt_turn<4>(x, lane);
                        const int first = br - (lane & 7);
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            if (first + k < s.rows && col < a.vd)
                                *reinterpret_cast<uint4*>(piece + 2 * a.block + (size_t)(first + k) * a.vd + col) = make_uint4(x[k][0], x[k][1], x[k][2], x[k][3]);
                    }
                    __syncwarp();
                }
                if (mine && !it.whole && (!both || slot == 0)) {
                    reinterpret_cast<float2*>(piece)[br] = make_float2(m * a.scale2, l);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty);
            item++;
        }
    }
    __syncwarp();
    if (!ok && lane == 0) atomicExch(a.error_flag, DETB_ERR_WAIT_EXPIRED);
    copies_wait_all();
    tc_fence_before();
    __syncthreads();
    if (warp == PRODUCTS) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------------------------------ host side
void ftree_tc_shape(int rows, int kd, int vd, int* block, int* tile, int* turn) {
    const bool wide = kd > 128 || vd > 128;
    *block = wide || rows <= TT_ROWS ? TT_ROWS : 2 * TT_ROWS;
    *tile = wide ? 64 : 128;
    *turn = 4;
}

// A cache's keys or values (`size` elements a head) as [rows][heads][size], boxes of 64 elements of one head x `box` rows, zeros outside.
// Address and rows are the first cache's that the kernel sets; here they only have to be well formed.
static bool cache_map(CUtensorMap* map, const TreeArgs& a, int size, int box) {
    const cuuint64_t dims[3] = {(cuuint64_t)size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.cap};
    const cuuint64_t strides[2] = {(cuuint64_t)size * 2, (cuuint64_t)a.ld * 2};
    const cuuint32_t boxes[3] = {64, 1, (cuuint32_t)box}, estr[3] = {1, 1, 1};
    return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.maps, dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int SLOTS, int KT>
static cudaError_t launch(const TreeArgs& a, cudaStream_t q) {
    using Cfg = TtCfg<SLOTS, KT>;
    TtShape sh{};
    sh.nkb = (a.kd + 63) / 64;
    sh.nvb = (a.vd + 63) / 64;
    sh.q_bytes = sh.nkb * TT_ROWS * 128;
    sh.stage_bytes = std::max(sh.nkb, sh.nvb) * KT * 128;
    sh.twice = SLOTS == 2 && a.block == TT_ROWS;
    const size_t fixed = (size_t)SLOTS * sh.q_bytes + sizeof(TtTables);
    sh.stages = (int)std::min<size_t>(TT_STAGES, (TREE_SMEM - fixed) / sh.stage_bytes);
    const size_t smem = fixed + (size_t)sh.stages * sh.stage_bytes;
    const cudaError_t e = most_smem(k_ftree_tc<SLOTS, KT>);
    if (e != cudaSuccess) return e;
    CUtensorMap keys, values;
    if (!cache_map(&keys, a, a.kd, KT) || !cache_map(&values, a, a.vd, KT)) return cudaErrorInvalidValue;
    return launch_pdl_try(k_ftree_tc<SLOTS, KT>, dim3(a.ctas), dim3(Cfg::THREADS), smem, q, 1, keys, values, a, sh);
}

cudaError_t ftree_tc_launch(const TreeArgs& a, cudaStream_t q) { return a.tile == 128 ? launch<2, 128>(a, q) : launch<1, 64>(a, q); }

}  // namespace detb
