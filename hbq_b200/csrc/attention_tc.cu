// Attention of many rows against a cache on the tensor core (tcgen05), scores and weights in tensor memory.
//
// The G query heads of a key head and the rows of a sequence -- or, against a shared prefix, of all sequences -- form one
// left operand: row r is token r / G, head r % G.  A block takes 256 of its rows as two tiles of 128 and walks over tiles of
// 128 keys:  S = Q K^T into tensor memory;  one warpgroup per row tile (thread = row) reads its row of S, masks it, keeps
// the running maximum and sum of a softmax and writes the weights back over S in the values' type;  O += P V with P from tensor
// memory.  While one warpgroup works on its tile's scores the tensor core multiplies for the other.
// O stays in tensor memory; its rows are rescaled only when a row's maximum has grown by more than 2^8 in the weights
// since the last time (larger weights are as exact as weights up to 1, and the sum divides the factor out again).
//
// Keys come by TMA in a ring that keys and values share, from a cache of any strides.  Tiles that the masks of all rows hide
// are left out; the mask is applied only in tiles that hide some key from some row.  There the weights hold zeros, and a
// zero times an infinity or a NaN of a hidden value would still reach the sum: such values are set to zero in shared memory
// before the product, and the rows of such a block are given what they see of them at the end (give_specials).  An infinity of a tile
// that all rows see becomes a NaN where a row's weight rounds to zero: a row that ends with a NaN is looked into likewise.
//
// What bounds it: per pair of 128 x 128 tiles the products take 2048 cycles at heads of 128, and shared memory delivers their operands in
// as many; the powers of two take 2048 on the special-function unit, a quarter of which is computed on the FMA pipe instead.  A
// row tile's softmax (some 1700 cycles) and the products it waits for (1024 and 300 of hand-over) follow one another, since the weights
// lie on the scores: tensor memory has no room for both.  The tensor pipe is busy 51 to 53 % of the time.  8192 tokens, 32 / 8 heads of
// 128, bf16, 20 calls in a row: all keys 459 us, 1197 TFLOP/s; window of 4096 374 us, 1103 of visible pairs; under a sustained
// load, where the power cap holds the clock at 1.65 to 1.67 GHz, 442 to 453 us.  A block of one key tile takes some 7 us.
#include "attention_dev.cuh"
#include "tc_dev.cuh"

namespace hbq {

namespace {

constexpr int TILE = 128, TCT = 320;
constexpr uint32_t POLLS = 1u << 20;

template <int DP> struct TcShape {
    static constexpr int HALVES = DP / 64;
    static constexpr int STAGE = TILE * DP * 2, Q = 2 * TILE * DP * 2;
    static constexpr int NS = DP == 128 ? 5 : 8;
    static constexpr int BYTES = 1024 + Q + NS * STAGE + 256;
};

struct TcTask {
    uint32_t R;                        // rows of a key head: L * G, or B * L * G against a prefix
    int prefix, k_by_head, k_by_seq, v_by_head, v_by_seq, vector_out, tma_out;
};

// Bounded waits of one thread and of a warp.  One thread waits for, issues and commits the products (a warp whose lanes vote on each
// wait: 944 -> 1024 TFLOP/s with 8192 tokens, all keys); the rows' warps poll with all lanes (lane 0 and a shuffle: 606
// and 536 us).
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code)
{
    #pragma unroll 1
    for (uint32_t it = 0; it < POLLS; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 63u && *abort_flag) return false;
    }
    *abort_flag = 1;
    atomicCAS(&g_tc_status, 0, code);
    return false;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code)
{
    #pragma unroll 1
    for (uint32_t it = 0; it < POLLS; ++it) {
        if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
        if ((it & 63u) == 63u && __any_sync(0xFFFFFFFFu, *abort_flag != 0)) return false;
    }
    if ((threadIdx.x & 31) == 0) { *abort_flag = 1; atomicCAS(&g_tc_status, 0, code); }
    __syncwarp();
    return false;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
// A warp's 32 rows from shared memory, once every lane has written its own (whole warp)
__device__ __forceinline__ void rows_written()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}
__device__ __forceinline__ void store_rows(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3)
{
    rows_written();
    if ((threadIdx.x & 31) == 0)
        asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];\n cp.async.bulk.commit_group;"
                     ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void store_parts(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3, int c4)
{
    rows_written();
    if ((threadIdx.x & 31) == 0)
        asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];\n cp.async.bulk.commit_group;"
                     ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4) : "memory");
}
// The stores so far have read their memory (whole warp)
__device__ __forceinline__ void rows_read()
{
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// Values [keys][64 columns of a head] with 128-byte rows and 128-byte swizzle, as the right operand whose rows are keys
// (the contraction): 8 keys 1024 B apart, 64 columns one half tile apart.
__device__ __forceinline__ uint64_t values_desc(uint32_t saddr)
{
    constexpr uint32_t kHi = 64u | (1u << 14) | (2u << 29);
    constexpr uint32_t kLbo = (TILE * 128) >> 4;
    return ((uint64_t)kHi << 32) | ((saddr & 0x3FFFFu) >> 4) | (kLbo << 16);
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1)
{
    asm("{ .reg .b64 ra, rb;\n mov.b64 ra, {%0, %1};\n mov.b64 rb, {%2, %3};\n add.rn.f32x2 ra, ra, rb;\n mov.b64 {%0, %1}, ra; }"
        : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1));
}

// Two powers of two on the FMA pipe (the special-function unit alone would take as long as the products): x = n + f with
// n the nearest whole number, 2^f by a polynomial on [-1/2, 1/2] (minimax in the relative error, 2.7e-6), 2^n from its bits.
// n is at least -127, whose bits are those of 0; a NaN stays one.
__device__ __forceinline__ void exp2_pair(float& x, float& y)
{
    constexpr float MAGIC = 12582912.f + 127.f;                // 1.5 * 2^23: the sum's last bits are n + 127
    constexpr float C0 = 0.9999992847f, C1 = 0.6931217909f, C2 = 0.2402474433f, C3 = 0.0559178628f, C4 = 0.00957010221f;
    float t0, t1, p0, p1;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(-127.f));
    asm("{ .reg .b64 x, t, r, f, p, k;\n"
        " mov.b64 x, {%4, %5};\n mov.b64 k, {%6, %6};\n add.rn.f32x2 t, x, k;\n mov.b64 {%0, %1}, t;\n"
        " mov.b64 k, {%7, %7};\n add.rn.f32x2 r, t, k;\n mov.b64 k, {%8, %8};\n fma.rn.f32x2 f, r, k, x;\n"
        " mov.b64 p, {%9, %9};\n mov.b64 k, {%10, %10};\n fma.rn.f32x2 p, p, f, k;\n mov.b64 k, {%11, %11};\n fma.rn.f32x2 p, p, f, k;\n"
        " mov.b64 k, {%12, %12};\n fma.rn.f32x2 p, p, f, k;\n mov.b64 k, {%13, %13};\n fma.rn.f32x2 p, p, f, k;\n mov.b64 {%2, %3}, p; }"
        : "=&f"(t0), "=&f"(t1), "=&f"(p0), "=&f"(p1)
        : "f"(x), "f"(y), "f"(MAGIC), "f"(-MAGIC), "f"(-1.f), "f"(C4), "f"(C3), "f"(C2), "f"(C1), "f"(C0));
    x = p0 * __uint_as_float(__float_as_uint(t0) << 23);
    y = p1 * __uint_as_float(__float_as_uint(t1) << 23);
}

template <class E> struct Word;
template <> struct Word<__half> {
    static constexpr uint32_t FORMAT = 0, INF = 0x7C00u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return h2_bits(__floats2half2_rn(a, b)); }
    static __device__ __forceinline__ float up(uint16_t u) { return __half2float(bits_h(u)); }
};
template <> struct Word<__nv_bfloat16> {
    static constexpr uint32_t FORMAT = 1, INF = 0x7F80u;
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float up(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
};

// The first n bits
__device__ __forceinline__ uint32_t first_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

// What the rows of a block see, in key positions: all rows that see anything stand between pa and pb.
struct Span {
    int pa, pb, window, sinks;         // window: 0 for none
    int first_tiles, low_tile;         // list of key tiles: the first `first_tiles` ones, then those from low_tile on
    int count;
    __device__ __forceinline__ int tile(int u) const { return u < first_tiles ? u : low_tile + u - first_tiles; }
    // every key of the tile is seen by every row between pa and pb
    __device__ __forceinline__ bool whole(int j0) const
    {
        return j0 + TILE - 1 <= pa && (window == 0 || j0 > pb - window || j0 + TILE - 1 < sinks);
    }
    __device__ __forceinline__ bool seen_by_some(int j) const { return j <= pb && (window == 0 || j > pa - window || j < sinks); }
};

// Puts the infinities and NaNs that row (b, i) of each `wanted` lane sees, of the prefix or of its own keys, into 32 columns (from d0 on) of
// its sums in tensor memory.  By a whole warp, out of line, past the SM's own cache (begin_beside).  The keys that all wanted
// rows see are shared out among the lanes, the rest of a row's are its lane's (a lane for all of its row's: 56 ms for 8192
// tokens in place of 4).  Of all keys for a piece of them too: the pieces' sum is what it is in each.
template <class E>
__device__ __noinline__ void give_specials(const AttnArgs& a, int prefix, uint32_t b, uint32_t i, uint32_t hk, int d0, bool wanted, uint32_t sums)
{
    constexpr uint32_t INF = Word<E>::INF, EXPONENTS = INF * 0x10001u, ONE = (0x8000u - INF) * 0x10001u;
    const uint16_t* v = (prefix ? static_cast<const uint16_t*>(a.pv) + (int64_t)hk * a.pvs[0]
                                : static_cast<const uint16_t*>(a.v) + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[1]) + d0;
    const int64_t step = prefix ? a.pvs[1] : a.vs[2];
    int lo = 0, end = 0, first = 0;                          // this row's keys: those before `first`, and lo .. end - 1
    if (wanted) {
        int64_t n, p;
        sequence_of(a, b, &n, &p);
        p += i;
        lo = !prefix && a.window > 0 && p >= a.window ? (int)(p - a.window + 1) : 0;
        end = prefix ? (int)a.P : (int)p + 1;
        first = a.sinks < lo ? (int)a.sinks : lo;
    }
    int all_lo = __reduce_max_sync(0xFFFFFFFFu, lo), all_end = __reduce_min_sync(0xFFFFFFFFu, wanted ? end : 0x7FFFFFFF);
    const int all_first = __reduce_min_sync(0xFFFFFFFFu, wanted ? first : 0x7FFFFFFF);
    if (all_lo >= all_end) all_lo = all_end = 0x7FFFFFFF;    // nothing in common
    const int lane = threadIdx.x & 31;
    uint32_t above = 0, below = 0;                           // a bit a column: infinities; NaNs are in both
    #pragma unroll 1
    for (int run = 0; run < 5; ++run) {
        if (run == 2) {
            above = __reduce_or_sync(0xFFFFFFFFu, above);
            below = __reduce_or_sync(0xFFFFFFFFu, below);
        }
        const int n = run < 2 ? 32 : 1;
        const int j0 = run == 0 ? lane : run == 1 ? (all_lo < all_end ? all_lo + lane : 0) : run == 2 ? all_first : run == 3 ? lo : max(all_end, lo);
        const int j1 = run == 0 ? all_first : run == 1 ? (all_lo < all_end ? all_end : 0) : run == 2 ? first : run == 3 ? min(all_lo, end) : end;
        #pragma unroll 1
        for (int64_t j = j0; j < j1 && (above & below) != 0xFFFFFFFFu; j += 2 * n) {
            uint4 x[8];                                      // two keys' four pieces of eight columns
            #pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int64_t key = j + (c >> 2) * n;
                x[c] = make_uint4(0, 0, 0, 0);
                if (key < j1 && d0 + 8 * (c & 3) < (int)a.D) x[c] = __ldcg(reinterpret_cast<const uint4*>(v + key * step + 8 * (c & 3)));
            }
            #pragma unroll
            for (int c = 0; c < 8; ++c) {
                // (an exponent of ones and one more sets the bit above it)
                if (!((((x[c].x & EXPONENTS) + ONE) | ((x[c].y & EXPONENTS) + ONE) | ((x[c].z & EXPONENTS) + ONE) | ((x[c].w & EXPONENTS) + ONE)) & 0x80008000u)) continue;
                #pragma unroll 1
                for (int e = 0; e < 8; ++e) {
                    const uint32_t u = (e < 4 ? (e < 2 ? x[c].x : x[c].y) : e < 6 ? x[c].z : x[c].w) >> (16 * (e & 1)) & 0xFFFFu, bit = 1u << (8 * (c & 3) + e);
                    if ((u & INF) != INF) continue;
                    const bool is_nan = (u & 0x7FFFu) != INF;
                    if (is_nan || u < 0x8000u) above |= bit;
                    if (is_nan || u >= 0x8000u) below |= bit;
                }
            }
        }
        __syncwarp();
    }
    float o[32];
    tc_ld32(sums, o);
    uint32_t w[32];
    #pragma unroll
    for (int e = 0; e < 32; ++e) {
        const bool p = wanted && ((above >> e) & 1u), m = wanted && ((below >> e) & 1u);
        w[e] = p && m ? 0x7FFFFFFFu : p ? 0x7F800000u : m ? 0xFF800000u : __float_as_uint(o[e]);
    }
    tc_st16(sums, w);
    tc_st16(sums + 16, w + 16);
    tc_st_wait();
}

template <class E, int DP>
__global__ void __launch_bounds__(TCT, 1) attention_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                              const __grid_constant__ CUtensorMap map_o,
                                                              const __grid_constant__ AttnArgs a, const __grid_constant__ TcTask task)
{
    using Sh = TcShape<DP>;
    constexpr float SHIFT = Weights<E>::SHIFT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t qs = base, ring = base + Sh::Q, ctrl = ring + Sh::NS * Sh::STAGE;
    uint8_t* ctrl_p = smem_raw + (ctrl - raw);
    const uint32_t kv_full = ctrl, kv_empty = ctrl + 8 * Sh::NS, q_full = ctrl + 16 * Sh::NS;
    const uint32_t s_full = q_full + 8, p_ready = q_full + 24, o_full = q_full + 40;        // two each
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl_p + 16 * Sh::NS + 64);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl_p + 16 * Sh::NS + 72);
    volatile int* special = reinterpret_cast<volatile int*>(ctrl_p + 16 * Sh::NS + 76);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Sh::NS; ++s) { mbar_init(kv_full + 8 * s, 1); mbar_init(kv_empty + 8 * s, 1); }
        mbar_init(q_full, 8);
        for (int t = 0; t < 2; ++t) { mbar_init(s_full + 8 * t, 1); mbar_init(p_ready + 8 * t, 4); mbar_init(o_full + 8 * t, 1); }
        *abort_flag = 0;
        *special = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    begin_beside(a);
    const uint32_t tmem = *tmem_slot;

    // this block: rows r0 .. r0 + 255 of key head hk of a sequence (group), a piece of their keys; the rows that see the
    // most keys first, so that the last blocks to start are short ones
    const uint32_t hk = blockIdx.x / (uint32_t)a.nsplit, split = blockIdx.x - hk * a.nsplit, group = blockIdx.y;
    const uint32_t r0 = (gridDim.z - 1 - blockIdx.z) * 256u, rend = min(r0 + 256u, task.R);
    const bool two = r0 + TILE < task.R;

    int64_t n64 = 0, first = 0;
    Span sp = {};
    sp.sinks = (int)min(a.sinks, (int64_t)0x7FFFFFFF);
    if (task.prefix) {
        sp.pa = sp.pb = (int)a.P - 1;
        sp.count = (int)((a.P + TILE - 1) / TILE);
    } else {
        sequence_of(a, group, &n64, &first);
        const int64_t p0 = first + r0 / a.G, p1 = first + (rend - 1) / a.G;
        const int64_t pa = p0 > 0 ? p0 : 0, pb = p1 < n64 - 1 ? p1 : n64 - 1;
        if (pa <= pb) {
            sp.pa = (int)pa; sp.pb = (int)pb;
            sp.window = a.window > 0 && a.window <= pb ? (int)a.window : 0;
            const int low = sp.window && sp.pa - sp.window + 1 > 0 ? sp.pa - sp.window + 1 : 0;
            sp.low_tile = low / TILE;
            const int st = sp.window ? (sp.sinks >= low ? sp.low_tile : (sp.sinks + TILE - 1) / TILE) : 0;
            sp.first_tiles = min(st, sp.low_tile);
            sp.count = sp.first_tiles + sp.pb / TILE - sp.low_tile + 1;
        }
    }
    // (a piece's tiles: counts times pieces stay below 2^31, keys being fewer than 2^31 and pieces 64)
    const int u0 = a.nsplit == 1 ? 0 : (int)((uint32_t)sp.count * split / (uint32_t)a.nsplit);
    const int u1 = a.nsplit == 1 ? sp.count : (int)((uint32_t)sp.count * (split + 1) / (uint32_t)a.nsplit), nt = u1 - u0;

    if (warp == 9) {
        // ================= keys and values =================
        if (lane == 0 && nt > 0) {
            const int kh = task.k_by_head ? (int)hk : 0, kb = task.k_by_seq ? (int)group : 0;
            const int vh = task.v_by_head ? (int)hk : 0, vb = task.v_by_seq ? (int)group : 0;
            uint32_t stage = 0, phase = 1;
            bool ok = true;
            for (int x = 0; x < 2 * nt && ok; ++x) {
                if (!(ok = wait_one(kv_empty + 8 * stage, phase, abort_flag, 41))) break;
                const int j0 = sp.tile(u0 + (x >> 1)) * TILE;
                const uint32_t dst = ring + stage * Sh::STAGE, bar = kv_full + 8 * stage;
                mbar_expect_tx(bar, Sh::STAGE);
                #pragma unroll
                for (int h = 0; h < Sh::HALVES; ++h) {
                    if (x & 1) tma_load_4d(dst + h * (TILE * 128), &map_v, h * 64, j0, vh, vb, bar);
                    else tma_load_4d(dst + h * (TILE * 128), &map_k, h * 64, j0, kh, kb, bar);
                }
                if (++stage == Sh::NS) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 8) {
        // ================= products =================
        if (nt > 0 && elect_one()) {
            constexpr uint32_t S_IDESC = (1u << 4) | (Word<E>::FORMAT << 7) | (Word<E>::FORMAT << 10) | ((TILE >> 3) << 17) | ((TILE >> 4) << 24);
            constexpr uint32_t O_IDESC = (1u << 4) | (Word<E>::FORMAT << 7) | (Word<E>::FORMAT << 10) | (1u << 16) | ((DP >> 3) << 17) | ((TILE >> 4) << 24);
            auto scores = [&](int t, uint32_t stage) {
                const uint32_t ka = ring + stage * Sh::STAGE, qa = qs + t * (TILE * 128);
                #pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    tc_mma_f16(tmem + t * TILE, umma_desc(qa + (kk >> 2) * (2 * TILE * 128) + (kk & 3) * 32),
                               umma_desc(ka + (kk >> 2) * (TILE * 128) + (kk & 3) * 32), S_IDESC, kk != 0);
                tc_commit(s_full + 8 * t);
            };
            auto output = [&](int t, uint32_t stage, bool more) {
                const uint32_t va = ring + stage * Sh::STAGE;
                #pragma unroll
                for (int kk = 0; kk < TILE / 16; ++kk)
                    mma_ts(tmem + 2 * TILE + t * DP, tmem + t * TILE + kk * 8, values_desc(va + kk * 2048), O_IDESC, more || kk != 0);
            };
            uint32_t ks = 0, kph = 0;                       // stage and phase of the next ring entry
            auto next = [&] { if (++ks == Sh::NS) { ks = 0; kph ^= 1u; } };
            bool ok = wait_one(q_full, 0, abort_flag, 42) && wait_one(kv_full + 8 * ks, kph, abort_flag, 43);
            if (ok) {
                tc_fence_after();
                scores(0, ks);
                if (two) scores(1, ks);
                tc_commit(kv_empty + 8 * ks);
                next();
            }
            for (int j = 0; j < nt && ok; ++j) {
                const uint32_t vs = ks, par = (uint32_t)j & 1u;
                const bool more = j + 1 < nt;
                if (!(ok = wait_one(kv_full + 8 * ks, kph, abort_flag, 43))) break;
                next();
                if (!(ok = wait_one(p_ready, par, abort_flag, 44))) break;
                tc_fence_after();
                output(0, vs, j > 0);
                if (more) {
                    if (!(ok = wait_one(kv_full + 8 * ks, kph, abort_flag, 43))) break;
                    tc_fence_after();
                    scores(0, ks);
                } else tc_commit(o_full);
                if (two) {
                    if (!(ok = wait_one(p_ready + 8, par, abort_flag, 44))) break;
                    tc_fence_after();
                    output(1, vs, j > 0);
                }
                if (more) {                                  // (behind the last values nothing is loaded)
                    tc_commit(kv_empty + 8 * vs);
                    if (two) scores(1, ks);
                    tc_commit(kv_empty + 8 * ks);
                    next();
                } else if (two) tc_commit(o_full + 8);
            }
        }
    } else {
        // ================= rows =================
        const int t = warp >> 2, wr = (warp & 3) * 32 + lane;
        // sequence, token and head of the thread's row; found again for the results, not kept: the loop needs every register
        const auto row_at = [&](uint32_t r, uint32_t& b, uint32_t& i, uint32_t& h) {
            asm volatile("" : "+r"(r));
            b = group;
            if (task.prefix) { b = r / (a.L * a.G); r -= b * (a.L * a.G); }
            i = r / a.G;
            h = hk * a.G + (r - i * a.G);
        };
        int hi = -1, lo = 0;                                 // this row sees keys lo .. hi and those before sp.sinks
        int64_t at = -1;                                     // its queries
        if (r0 + t * TILE + wr < rend) {
            uint32_t b, i, h;
            row_at(r0 + t * TILE + wr, b, i, h);
            at = (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)h * a.qs[2];
            if (task.prefix) sequence_of(a, b, &n64, &first);
            const int64_t p = first + i;
            if (p < n64) {
                if (task.prefix) hi = (int)a.P - 1;
                else if (p >= 0) {
                    hi = (int)p;
                    lo = sp.window ? (int)p - sp.window + 1 : 0;
                }
            }
        }
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_col = lanes + t * TILE, o_col = s_col + 2 * TILE + t * (DP - TILE);
        bool ok = true;
        float m = -INFINITY, l = 0.f;
        const float c = a.scale_log2;
        if (nt > 0) {
            // queries of this warp's 32 rows: 16-byte pieces, neighbouring lanes along a row, all on their way at once; a row's
            // address comes from the lane that owns the row.  (Little code, too: what a block runs once it fetches cold.)
            constexpr int PIECES = DP / 8;
            const int pc = lane % PIECES, own = lane / PIECES;
            #pragma unroll 4
            for (int k = 0; k < PIECES; ++k) {
                const int64_t from = __shfl_sync(0xFFFFFFFFu, at, k * (32 / PIECES) + own);
                const bool in = from >= 0 && pc * 8 < (int)a.D;
                const E* p = static_cast<const E*>(a.q) + (in ? from + pc * 8 : 0);
                const uint32_t q = warp * 32 + k * (32 / PIECES) + own;
                const uint32_t dst = qs + (pc >> 3) * (2 * TILE * 128) + q * 128 + (((pc & 7) ^ (q & 7)) * 16);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p), "r"(in ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        uint32_t vs = 1, vph = 0;                            // ring entry of this step's values
        if (t == 0 || two)
        for (int u = 0; u < nt; ++u) {
            const int j0 = sp.tile(u0 + u) * TILE;
            const bool whole = sp.whole(j0);
            if (!whole && t == 0) {
                // infinities and NaNs among this tile's values, while the scores are on their way: thread = key
                if (!(ok = wait_for(kv_full + 8 * vs, vph, abort_flag, 46))) break;
                const uint32_t row = ring + vs * Sh::STAGE + wr * 128;
                constexpr uint32_t EXPONENTS = Word<E>::INF * 0x10001u, ONE = (0x8000u - Word<E>::INF) * 0x10001u;
                bool found = false;
                #pragma unroll
                for (int pc = 0; pc < DP / 8; ++pc) {
                    const uint32_t at = row + (pc >> 3) * (TILE * 128) + (((pc & 7) ^ (wr & 7)) * 16);
                    uint32_t v[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
                    uint32_t bad = 0;                        // (an exponent of ones and one more sets the bit above it)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) bad |= (v[e] & EXPONENTS) + ONE;
                    if (bad & 0x80008000u) found = true;
                }
                if (found) {
                    if (sp.seen_by_some(j0 + wr)) { *special = 1; __threadfence_block(); }
                    #pragma unroll 1
                    for (int pc = 0; pc < DP / 8; ++pc) {
                        const uint32_t at = row + (pc >> 3) * (TILE * 128) + (((pc & 7) ^ (wr & 7)) * 16);
                        #pragma unroll 1
                        for (int e = 0; e < 4; ++e) {
                            uint32_t v;
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at + 4 * e) : "memory");
                            if ((v & Word<E>::INF) == Word<E>::INF) v &= 0xFFFF0000u;
                            if ((v & (Word<E>::INF << 16)) == (Word<E>::INF << 16)) v &= 0x0000FFFFu;
                            asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 4 * e), "r"(v) : "memory");
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
            }
            if (!(ok = wait_for(s_full + 8 * t, (uint32_t)u & 1u, abort_flag, 45))) break;
            tc_fence_after();
            uint32_t s[128];
            #pragma unroll
            for (int k = 0; k < 4; ++k) tc_ld32_issue(s_col + 32 * k, s + 32 * k);
            tc_ld_wait(s);
            #pragma unroll
            for (int k = 1; k < 4; ++k) tc_ld_landed(s + 32 * k);
            if (!whole) {
                #pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int k0 = j0 + 32 * q;
                    const uint32_t seen = first_bits(hi + 1 - k0) & (~first_bits(lo - k0) | first_bits(sp.sinks - k0));
                    #pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!(seen & (1u << k))) s[32 * q + k] = 0xFF800000u;
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            #pragma unroll
            for (int k = 0; k < 128; k += 2)
                asm("max.f32 %0, %0, %1, %2;" : "+f"(mx[(k >> 1) & 3]) : "f"(__uint_as_float(s[k])), "f"(__uint_as_float(s[k + 1])));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const bool grow = (top - m) * c > GROWTH;        // (from -inf: any; -inf itself: NaN, false)
            if (__any_sync(0xFFFFFFFFu, grow)) {
                const float f = grow ? factor_of((m - top) * c) : 1.f;
                if (grow) m = top;
                l *= f;
                if (u > 0) {
                    #pragma unroll 1
                    for (int k = 0; k < DP / 16; ++k) {
                        uint32_t o[16];
                        asm volatile(
                            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                            "tcgen05.wait::ld.sync.aligned;"
                            : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]),
                              "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15]) : "r"(o_col + 16 * k) : "memory");
                        #pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tc_st16(o_col + 16 * k, o);
                    }
                }
            }
            const float off = SHIFT - (m == -INFINITY ? 0.f : m * c);
            float sum[4] = {};
            #pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t w[16];
                #pragma unroll
                for (int k = 0; k < 16; ++k) {
                    float x, y;
                    fma2(x, y, __uint_as_float(s[32 * q + 2 * k]), __uint_as_float(s[32 * q + 2 * k + 1]), c, off);
                    if ((k & 3) == 3) exp2_pair(x, y);          // a quarter of them
                    else { x = exp2_fast(x); y = exp2_fast(y); }
                    w[k] = Word<E>::pack(x, y);
                    add2(sum[2 * (k & 1)], sum[2 * (k & 1) + 1], x, y);
                }
                tc_st16(s_col + 16 * q, w);
            }
            vs += 2;
            if (vs >= Sh::NS) { vs -= Sh::NS; vph ^= 1u; }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tc_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready + 8 * t);
        }
        // ---- the rows' results ----
        if (ok && (t == 0 || two)) {
            if (nt > 0) ok = wait_for(o_full + 8 * t, 0, abort_flag, 47);
            tc_fence_after();
            const bool direct = a.parts == 0, add = nt > 0 && *special;
            const bool live = hi >= 0 && l != 0.f;            // (a NaN counts as something)
            const float f = direct ? (live ? 1.f / l : 0.f) : 1.f;
            const uint32_t r = r0 + t * TILE + wr;
            uint32_t b, i, h;
            row_at(r, b, i, h);
            const int64_t row = ((int64_t)b * a.L + i) * a.H + h;
            if (ok) {
                // Results leave by TMA where the warp's 32 rows are whole tokens (map_o: G heads by 32 / G tokens): each lane puts its
                // row into this row tile's queries' memory, which no product reads any more.  Stores of a row a lane touch 32 lines at
                // a time (4000 cycles a block).
                const uint32_t region = qs + warp * 4096;              // 32 rows of 128 bytes; the next 64 columns' lie 2 * TILE rows on
                const auto stage_in = [&](uint32_t at, int pc, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + lane * 128 + ((pc ^ (lane & 7)) * 16)), "r"(w0), "r"(w1), "r"(w2), "r"(w3) : "memory");
                };
                const uint32_t base_row = r0 + warp * 32;
                const int token = (int)(base_row / a.G), seq = task.prefix ? 0 : (int)group;
                const bool by_tma = task.tma_out && base_row < rend;   // (rows behind the last: nothing)
                #pragma unroll 1
                for (int k = 0; k < DP / 32; ++k) {
                    float o[32];
                    __syncwarp();
                    if (nt > 0) tc_ld32(o_col + 32 * k, o);
                    // (chains of maxima find a NaN with half the instructions of 32 comparisons: short prompts 29.6 -> 28.7 us)
                    float nan[4] = {o[28], o[29], o[30], o[31]};
                    #pragma unroll
                    for (int e = 0; e < 28; e += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(nan[(e >> 1) & 3]) : "f"(o[e]), "f"(o[e + 1]));
                    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(nan[0]) : "f"(nan[1]), "f"(nan[2]));
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(nan[0]) : "f"(nan[3]));
                    const bool look = live && l == l && (add || nan[0] != nan[0]);
                    if (__builtin_expect(__any_sync(0xFFFFFFFFu, look), 0)) {
                        give_specials<E>(a, task.prefix, b, i, hk, 32 * k, look, o_col + 32 * k);
                        tc_ld32(o_col + 32 * k, o);
                    }
                    if (!live) {
                        #pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.f;
                    }
                    if (direct) {
                        uint32_t w[16];
                        #pragma unroll
                        for (int z = 0; z < 16; ++z) w[z] = Word<E>::pack(o[2 * z] * f, o[2 * z + 1] * f);
                        if (by_tma) {
                            const uint32_t at = region + (k >> 1) * (2 * TILE * 128);
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) stage_in(at, 4 * (k & 1) + e, w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                            if (k & 1) store_rows(&map_o, at, 64 * (k >> 1), (int)(hk * a.G), token, seq);
                        } else if (r < rend) {
                            uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)b * a.os[0] + (int64_t)i * a.os[1] + (int64_t)h * a.os[2] + 32 * k;
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (32 * k + 8 * e >= (int)a.D) break;
                                if (task.vector_out) *reinterpret_cast<uint4*>(out + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                                else {
                                    #pragma unroll
                                    for (int z = 0; z < 8; ++z) out[8 * e + z] = (uint16_t)(w[4 * e + (z >> 1)] >> (16 * (z & 1)));
                                }
                            }
                        }
                    } else if (by_tma) {
                        const uint32_t at = region + (k & (DP / 64 - 1)) * (2 * TILE * 128);
                        if (k >= DP / 64 && (k & (DP / 64 - 1)) == 0) rows_read();
                        #pragma unroll
                        for (int e = 0; e < 8; ++e)
                            stage_in(at, e, __float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]), __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3]));
                        store_parts(&map_o, at, 32 * k, a.part0 + (int)split, (int)(hk * a.G), token, seq);
                    } else if (r < rend) {
                        float* part = part_sum(a, row, a.part0 + split);
                        #pragma unroll
                        for (int e = 0; e < 32; e += 8)          // whole sectors
                            if (32 * k + e < (int)a.D)
                                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(part + 32 * k + e), "f"(o[e]), "f"(o[e + 1]),
                                             "f"(o[e + 2]), "f"(o[e + 3]), "f"(o[e + 4]), "f"(o[e + 5]), "f"(o[e + 6]), "f"(o[e + 7]) : "memory");
                    }
                }
                if (by_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
                if (!direct && r < rend)
                    *part_weight(a, row, a.part0 + split) = live ? make_float2((m == -INFINITY ? 0.f : m * c) - SHIFT, l) : make_float2(-INFINITY, 0.f);
            }
        }
    }

    // ---- teardown: every role arrives here, also after an expired wait ----
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // let copies that may still be in flight land before the block's shared memory is released
        const unsigned long long t0 = gtime_ns();
        while (gtime_ns() - t0 < 200000ull) { }
        __syncthreads();
    }
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    end_beside(a);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder()
{
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qr;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) == cudaSuccess && qr == cudaDriverEntryPointSuccess;
        return ok ? (EncodeFn)p : (EncodeFn) nullptr;
    }();
    return fn;
}

int encode(CUtensorMap* map, CUtensorMapDataType type, uint32_t rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box)
{
    EncodeFn fn = encoder();
    if (!fn) return HBQ_ERR_CUDA;
    const cuuint32_t each[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, type, rank, const_cast<void*>(ptr), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? HBQ_OK : HBQ_ERR_CUDA;
}
// The output [sequence][token][head][D] in boxes of G heads by 32 / G tokens; against a prefix the sequences' tokens are one
// axis, where their steps allow it.
int out_map(CUtensorMap* map, const AttnArgs& a, int dtype, bool prefix)
{
    if (prefix && a.L > 1 && a.B > 1 && a.os[0] != (int64_t)a.L * a.os[1]) return HBQ_ERR_UNSUPPORTED;
    const int64_t tokens = prefix ? (int64_t)a.B * a.L : a.L, step = prefix && a.L == 1 ? a.os[0] : a.os[1];
    const auto bytes = [&](int64_t stride) { return (cuuint64_t)(stride > 0 ? stride : a.D) * 2; };      // (an axis of one element has any step)
    const cuuint64_t dims[4] = {a.D, a.H, (cuuint64_t)tokens, prefix ? 1u : a.B}, strides[3] = {bytes(a.os[2]), bytes(step), bytes(a.os[0])};
    const cuuint32_t box[4] = {64, a.G, 32 / a.G, 1};
    return encode(map, dtype == HBQ_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, a.out, dims, strides, box);
}
// The rows' lists of parts [sequence][token][head][part][D], likewise
int parts_map(CUtensorMap* map, const AttnArgs& a, bool prefix)
{
    const cuuint64_t list = (cuuint64_t)a.parts * a.D * 4, token = list * a.H, tokens = prefix ? (cuuint64_t)a.B * a.L : a.L;
    const cuuint64_t dims[5] = {a.D, (cuuint64_t)a.parts, a.H, tokens, prefix ? 1u : a.B}, strides[4] = {a.D * 4ull, list, token, token * a.L};
    const cuuint32_t box[5] = {32, 1, a.G, 32 / a.G, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 5, a.part, dims, strides, box);
}

template <class E, int DP>
int tc_launch(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mo, const AttnArgs& a, const TcTask& task, dim3 blocks, cudaStream_t stream)
{
    { const int rc = ensure_dynamic_smem(attention_tc_kernel<E, DP>, TcShape<DP>::BYTES); if (rc) return rc; }
    HBQ_CUDA_TRY(launch_dependent(attention_tc_kernel<E, DP>, blocks, TCT, (size_t)TcShape<DP>::BYTES, stream, mk, mv, mo, a, task));
    HBQ_LAUNCH_CHECK("attention_tc_kernel");
    return HBQ_OK;
}

}  // namespace

// A cache [sequences][heads][keys][D] in boxes of `rows` keys by 64 values; keys beyond the last and values beyond D read as
// zeros.  An axis whose elements are all the same ones (stride 0) is left out.
int attention_cache_map(CUtensorMap* map, const void* ptr, int dtype, int64_t D, int rows, int64_t keys, int64_t key_stride, int64_t heads, int64_t head_stride,
              int64_t seqs, int64_t seq_stride)
{
    const auto step = [](int64_t stride, int64_t other) { return (cuuint64_t)(stride > 0 ? stride : other) * 2; };
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)keys, (cuuint64_t)(head_stride > 0 ? heads : 1), (cuuint64_t)(seq_stride > 0 ? seqs : 1)};
    const cuuint64_t strides[3] = {step(key_stride, D), step(head_stride, D), step(seq_stride, D)};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
    return encode(map, dtype == HBQ_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, ptr, dims, strides, box);
}

// Into how many pieces the keys of a block's rows are cut: the count with the shortest longest SM, where a block costs its
// key tiles and about three tiles' time to start and end, and joining pieces about four.
int attention_tc_parts(const hbq_attention* p, bool prefix)
{
    int sms = 148;
    device_sms(&sms);
    const int64_t G = p->H / p->Hkv, R = (prefix ? p->B : 1) * p->L * G, blocks = (R + 255) / 256 * p->Hkv * (prefix ? 1 : p->B);
    int64_t keys = prefix ? p->P : p->S;
    if (!prefix && p->window > 0 && p->window + p->sinks + 256 / G + 256 < keys) keys = p->window + p->sinks + 256 / G + 256;
    const int64_t tiles = (keys + TILE - 1) / TILE;
    int64_t best = 1, cost = (blocks + sms - 1) / sms * (tiles + 3);
    for (int64_t n = 2; n <= 64 && n <= tiles && blocks * n <= 2 * sms; ++n) {
        const int64_t now = (blocks * n + sms - 1) / sms * ((tiles + n - 1) / n + 3) + 4;
        if (now < cost) { cost = now; best = n; }
    }
    return (int)best;
}

// The rows of `a` against their own keys, or (prefix) all sequences' rows against the prefix.
int attention_tc_launch(AttnArgs& a, int dtype, bool prefix, cudaStream_t stream)
{
    TcTask task = {};
    const int64_t R = (int64_t)(prefix ? a.B : 1) * a.L * a.G;
    if (R > 0x7FFFFF00ll) return HBQ_ERR_UNSUPPORTED;
    task.R = (uint32_t)R; task.prefix = prefix;
    const uint32_t tiles = (task.R + 255) / 256;
    if (tiles > 65535) return HBQ_ERR_UNSUPPORTED;                 // (sequences are at most that many by the call's checks)
    const dim3 blocks(a.Hkv * (unsigned)a.nsplit, prefix ? 1u : a.B, tiles);
    const int64_t pks[3] = {0, a.pks[0], a.pks[1]}, pvs[3] = {0, a.pvs[0], a.pvs[1]};
    const int64_t *ks = prefix ? pks : a.ks, *vs = prefix ? pvs : a.vs;
    task.k_by_seq = ks[0] > 0; task.k_by_head = ks[1] > 0; task.v_by_seq = vs[0] > 0; task.v_by_head = vs[1] > 0;
    task.vector_out = ((a.os[0] | a.os[1] | a.os[2]) % 8) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    CUtensorMap mk, mv, mo = {};
    if (32 % a.G == 0) {
        const int rc = a.parts ? parts_map(&mo, a, prefix) : task.vector_out ? out_map(&mo, a, dtype, prefix) : HBQ_ERR_UNSUPPORTED;
        if (rc && rc != HBQ_ERR_UNSUPPORTED) return rc;
        task.tma_out = rc == HBQ_OK;
    }
    const int64_t keys = prefix ? a.P : a.S;
    { const int rc = attention_cache_map(&mk, prefix ? a.pk : a.k, dtype, a.D, TILE, keys, ks[2], a.Hkv, ks[1], a.B, ks[0]); if (rc) return rc; }
    { const int rc = attention_cache_map(&mv, prefix ? a.pv : a.v, dtype, a.D, TILE, keys, vs[2], a.Hkv, vs[1], a.B, vs[0]); if (rc) return rc; }
    const bool wide = a.D > 64;
    if (dtype == HBQ_DTYPE_F16)
        return wide ? tc_launch<__half, 128>(mk, mv, mo, a, task, blocks, stream) : tc_launch<__half, 64>(mk, mv, mo, a, task, blocks, stream);
    return wide ? tc_launch<__nv_bfloat16, 128>(mk, mv, mo, a, task, blocks, stream)
                : tc_launch<__nv_bfloat16, 64>(mk, mv, mo, a, task, blocks, stream);
}

int attention_rows_status(int* host_out);   // attention_rows.cu: that kernel's own status word
int attention_rows_status_reset();

int attention_tc_status(int* host_out)
{
    HBQ_CUDA_TRY(cudaMemcpyFromSymbol(host_out, g_tc_status, sizeof(int)));
    return *host_out ? HBQ_OK : attention_rows_status(host_out);
}
int attention_tc_status_reset()
{
    const int z = 0;
    HBQ_CUDA_TRY(cudaMemcpyToSymbol(g_tc_status, &z, sizeof(int)));
    return attention_rows_status_reset();
}

}  // namespace hbq
