// Attention of few rows against a cache: the query heads that share a key head, for one token, on the warp-level MMA.
//
// For a row at position p the visible keys are the prefix, the first `sinks` ones and those behind p - window: three runs of
// the cache, walked over in steps of 16 keys.  Nothing that the mask hides enters the arithmetic: a run's last step may
// bring keys behind its end, whose scores become -inf and whose values zeros.  Bound by memory: keys and values are read once
// for up to 16 heads; one MMA tile is 16 rows by 8 keys, most of them empty for four heads, at a cost below the memory's.
//
// Each warp has a ring of its own, filled by TMA (one lane; with asynchronous copies by all lanes the addresses took most of
// the instructions, and the kernel was bound by their latency at 4.7 TB/s), a maximum, a weight and a sum of its own; no
// barrier until the warps' sums are joined at the end of a row group.  As in the tensor-core kernel the sums are rescaled only
// when a maximum has grown by more than 2^8 in the weights, so a step without that has no exchange between lanes.
//
// The lengths are known on the device alone and may be as different as one key and a hundred thousand.  So the row groups'
// units of 64 keys form one list over all sequences, of which every block takes an equal share; where a share
// begins or ends inside a group, its part (sum, maximum, weight) goes to a slot of the block and a second kernel joins.
// Where no group has many keys and there are few groups, a group belongs to a cluster of up to eight blocks instead, which join
// their parts through distributed shared memory: one launch, no workspace (one sequence of 1024 keys, 8 key heads: 10.8 -> 7.6 us
// in a graph).
//
// 32 sequences, 4100 visible keys each, 8 key heads of 128, bf16: 97 us, 5.6 TB/s (86 % of the measured copy rate); one of 131072
// keys 99 us; 8 of 8192 57 us, of which the data take 42: SMs do not get the memory's bandwidth in equal parts, and the last
// block ends at 54.
#include "attention_dev.cuh"
#include "tc_dev.cuh"
#include <type_traits>

namespace hbq {

namespace {

// Warps, stages a warp, keys a stage; 196 KB a SM in flight.  Two blocks of three stages: 96, 113 and 54 us (32 sequences of 4100 keys, one of
// 131072, 64 of 1024); three of two stages 96, 122 and 59; one of four 102, 106 and 66.
constexpr int RW = 4, STAGES = 3, GROUP = 16, BLOCKS_PER_SM = 2;
constexpr uint32_t POLLS = 1u << 20;

template <class E> struct Mma;
template <> struct Mma<__half> {
    static constexpr uint32_t ONES = 0x3C003C00u, INF = 0x7C00u;
    static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) { return h2_bits(__floats2half2_rn(x, y)); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(bits_h2(u)); }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) { static_cast<__half*>(p)[i] = __float2half_rn(v); }
};
template <> struct Mma<__nv_bfloat16> {
    static constexpr uint32_t ONES = 0x3F803F80u, INF = 0x7F80u;
    static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y)
    {
        __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) { static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); }
};

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int NK> struct RowsShape {
    static constexpr int DP = NK * 16;                       // head length, rounded up
    static constexpr int HALVES = (DP + 63) / 64, TILE = HALVES * GROUP * 128;       // 128-byte rows, swizzled by TMA
    static constexpr int STAGE = 2 * TILE;
    static constexpr int RING = RW * STAGES * STAGE;
    static constexpr int JOIN = RW * 16 * (DP + 2) * 4;
    static constexpr int BLOCK = 16 * (DP + 2) * 4;          // a cluster: this block's part
    static constexpr int BYTES = RING > JOIN + BLOCK ? RING : JOIN + BLOCK;
};

// The maps of a call's cache and prefix.
struct RowsMaps { CUtensorMap k, v, pk, pv; };

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_meet()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float at `addr` of the cluster's block `rank`
__device__ __forceinline__ float peer_load(uint32_t addr, uint32_t rank)
{
    float v;
    asm volatile("{ .reg .b32 p;\n mapa.shared::cluster.u32 p, %1, %2;\n ld.shared::cluster.f32 %0, [p]; }" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// The keys of row (b, i) in steps of 16: the prefix's, those of the first `ns` keys, those of keys lo .. p.
struct KeyList {
    int P, ns, lo, end;                                      // lengths of the first two runs; the third is lo .. end - 1
    int pre, sink, steps;                                    // steps of the first run, the first two, and all
};
__device__ __forceinline__ KeyList keys_of(const AttnArgs& a, uint32_t b, uint32_t i)
{
    int64_t n, p;
    sequence_of(a, b, &n, &p);
    p += i;
    KeyList k = {};
    if (p < n) {
        k.P = (int)a.P;
        if (p >= 0) {
            k.lo = a.window > 0 && p - a.window + 1 > 0 ? (int)(p - a.window + 1) : 0;
            k.ns = a.sinks < k.lo ? (int)a.sinks : k.lo;
            k.end = (int)p + 1;
        }
    }
    k.pre = k.P / GROUP + (k.P % GROUP != 0);
    k.sink = k.pre + k.ns / GROUP + (k.ns % GROUP != 0);
    k.steps = k.sink + (k.end - k.lo) / GROUP + ((k.end - k.lo) % GROUP != 0);
    return k;
}
// A group's units; one that sees nothing has one, in which its zeros are written.
__device__ __forceinline__ int64_t units_of(const KeyList& k) { return k.steps > RW ? (k.steps + RW - 1) / RW : 1; }

// Units before each token, [0 .. tokens], by the whole block (tokens at most two a thread).
__device__ void count_units(const AttnArgs& a, int64_t* table)
{
    __shared__ int64_t warps[RW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t tokens = a.B * a.L, r = 2 * threadIdx.x;
    int64_t c0 = 0, c1 = 0;
    if (r < tokens) c0 = units_of(keys_of(a, r / a.L, r % a.L));
    if (r + 1 < tokens) c1 = units_of(keys_of(a, (r + 1) / a.L, (r + 1) % a.L));
    int64_t sum = c0 + c1;
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int64_t below = __shfl_up_sync(0xFFFFFFFFu, sum, d);
        if (lane >= d) sum += below;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    int64_t before = sum - c0 - c1;
    for (int w = 0; w < warp; ++w) before += warps[w];
    if (r < tokens) { table[r] = before; table[r + 1] = before + c0; }
    if (r + 1 < tokens) table[r + 2] = before + c0 + c1;
    __syncthreads();
}

// (240 registers, as the walk that keeps infinities apart would like more: with 255 the kernel behind it finds no room beside it, 98.9 -> 100.6 us)
template <class E, int NK>
__global__ void __maxnreg__(240) attention_rows_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ RowsMaps maps, uint32_t tiles)
{
    using Sh = RowsShape<NK>;
    constexpr float SHIFT = Weights<E>::SHIFT;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ int64_t table[RW * 64 + 1];
    __shared__ __align__(8) uint64_t full[RW * STAGES];
    __shared__ int given_up;
    volatile int* abort_flag = &given_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int k = 0; k < RW * STAGES; ++k) mbar_init(smem_u32(&full[k]), 1);
        given_up = (smem_u32(smem) & 1023u) != 0;                    // (the copies' swizzle goes by address bits)
        if (given_up) atomicCAS(&g_tc_status, 0, 50);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    begin_beside(a);
    const uint32_t groups = a.Hkv * tiles, tokens = a.B * a.L;       // row groups of a token
    int64_t w0, w1, total = 1, takers = 1;                           // this block's share of the units
    uint32_t token;
    if (a.shared) {
        count_units(a, table);
        total = table[tokens] * groups;
        takers = rows_takers(a, total);
        if (blockIdx.x >= takers) { end_beside(a); return; }
        w0 = total * blockIdx.x / takers; w1 = total * (blockIdx.x + 1) / takers;
        uint32_t low = 0, high = tokens;                             // the last token that begins at or before w0
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (table[mid] * groups <= w0) low = mid; else high = mid;
        }
        token = low;
    } else {
        token = blockIdx.x / a.cluster / groups;
        w0 = 0; w1 = 1;
    }
    const int rank = a.shared ? 0 : (int)(blockIdx.x % a.cluster), stride = a.shared ? RW : RW * a.cluster;
    const uint32_t ring = smem_u32(smem) + warp * (STAGES * Sh::STAGE), bars = smem_u32(&full[warp * STAGES]);
    uint32_t stage = 0, phase = 0;                                   // the warp's next stage to read, and its parity
    bool ok = given_up == 0;
    while (w0 < w1) {
    const uint32_t b = token / a.L, i = token - b * a.L;
    const KeyList list = keys_of(a, b, i);
    int64_t take = 1;
    int x0 = 0, x1 = list.steps;                                     // this share's steps of the group
    uint32_t g;
    int slot = -1;                                                   // -1: the whole group
    if (a.shared) {
        const int64_t units = table[token + 1] - table[token], in = w0 - table[token] * groups;
        g = (uint32_t)(in / units);
        const int64_t off = in - g * units;
        take = min(units - off, w1 - w0);
        x0 = (int)off * RW;
        x1 = (int)min((int64_t)list.steps, (off + take) * RW);
        slot = take == units ? -1 : off > 0 ? 0 : 1;
        if (off == 0 && threadIdx.x == 0)
            a.table[(int64_t)token * groups + g] = make_int2(blockIdx.x, slot < 0 ? 0 : rows_owner(w0 + units - 1, total, takers) - (int)blockIdx.x + 1);
    } else g = blockIdx.x / a.cluster - token * groups;
    const uint32_t hk = g / tiles, g0 = (g - hk * tiles) * 16, rows = min(16u, a.G - g0), h0 = hk * a.G + g0;
    const int kh = a.ks[1] > 0 ? (int)hk : 0, kb = a.ks[0] > 0 ? (int)b : 0, vh = a.vs[1] > 0 ? (int)hk : 0, vb = a.vs[0] > 0 ? (int)b : 0;
    const int ph = a.pks[0] > 0 ? (int)hk : 0, pvh = a.pvs[0] > 0 ? (int)hk : 0;

    // one lane: step x into a stage
    auto load = [&](int x, uint32_t st) {
        const uint32_t dst = ring + st * Sh::STAGE, bar = bars + 8 * st;
        mbar_expect_tx(bar, Sh::STAGE);
        const bool pre = x < list.pre;
        const int j = pre ? x * GROUP : x < list.sink ? (x - list.pre) * GROUP : list.lo + (x - list.sink) * GROUP;
        #pragma unroll
        for (int h = 0; h < Sh::HALVES; ++h) {
            load_box(dst + h * (GROUP * 128), pre ? &maps.pk : &maps.k, h * 64, j, pre ? ph : kh, pre ? 0 : kb, bar);
            load_box(dst + Sh::TILE + h * (GROUP * 128), pre ? &maps.pv : &maps.v, h * 64, j, pre ? pvh : vh, pre ? 0 : vb, bar);
        }
    };
    const int first = x0 + rank * RW + warp;
    auto load_first = [&] {
        if (lane != 0 || !ok) return;
        uint32_t st = stage;
        for (int k = 0; k < STAGES && first + k * stride < x1; ++k) {
            load(first + k * stride, st);
            if (++st == STAGES) st = 0;
        }
    };
    load_first();

    // queries as the left operand's fragments: rows lane / 4 and lane / 4 + 8
    uint32_t qf[NK][4];
    #pragma unroll
    for (int kk = 0; kk < NK; ++kk)
        #pragma unroll
        for (int f = 0; f < 4; ++f) {
            const uint32_t r = lane / 4 + 8 * (f & 1), d = kk * 16 + (lane & 3) * 2 + 8 * (f >> 1);
            qf[kk][f] = r < rows && d < a.D
                ? __ldcg(reinterpret_cast<const unsigned*>(static_cast<const E*>(a.q) + (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)(h0 + r) * a.qs[2] + d)) : 0u;
        }

    float o[NK * 2][4], m[2], l[2];
    const float c = a.scale_log2;
    // The warp's steps.  A weight's second number may be zero or negative, and makes a NaN of an infinity among the values: `apart`
    // takes infinities and NaNs out of the products and multiplies them by one.
    const auto walk = [&](auto apart) {
        constexpr bool APART = decltype(apart)::value;
        #pragma unroll
        for (int t = 0; t < NK * 2; ++t)
            #pragma unroll
            for (int f = 0; f < 4; ++f) o[t][f] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
        for (int x = first; x < x1 && ok; x += stride) {
            {
                uint32_t it = 0;
                while (!__all_sync(0xFFFFFFFFu, mbar_try_wait(bars + 8 * stage, phase)))
                    if (++it == POLLS) { ok = false; break; }
                if (!ok) {
                    if (lane == 0) { *abort_flag = 1; atomicCAS(&g_tc_status, 0, 51); }
                    __syncwarp();
                    break;
                }
            }
            const uint32_t kt = ring + stage * Sh::STAGE, vt = kt + Sh::TILE;
            const int run = x < list.pre ? list.P - x * GROUP : x < list.sink ? list.ns - (x - list.pre) * GROUP : list.end - list.lo - (x - list.sink) * GROUP;
            if (run < GROUP) {                                           // values behind the run's end
                for (int y = lane; y < (GROUP - run) * Sh::HALVES * 8; y += 32) {
                    const int key = run + y / (Sh::HALVES * 8), pc = y % (Sh::HALVES * 8);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vt + (pc >> 3) * (GROUP * 128) + key * 128 + (pc & 7) * 16), "r"(0) : "memory");
                }
                __syncwarp();
            }
            float s[2][4] = {};
            #pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                uint32_t f[4];
                const int row = (lane & 7) + 8 * (lane >> 4), pc = (kk & 3) * 2 + ((lane >> 3) & 1);
                ldsm4(f, kt + (kk >> 2) * (GROUP * 128) + row * 128 + ((pc ^ (row & 7)) * 16));
                Mma<E>::run(s[0], qf[kk], f[0], f[1]);
                Mma<E>::run(s[1], qf[kk], f[2], f[3]);
            }
            if (run < GROUP) {
                #pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((e >> 2) * 8 + (lane & 3) * 2 + (e & 1) >= run) s[e >> 2][e & 3] = -INFINITY;
            }
            float top[2];
            #pragma unroll
            for (int r = 0; r < 2; ++r) top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            if (__any_sync(0xFFFFFFFFu, (top[0] - m[0]) * c > GROWTH || (top[1] - m[1]) * c > GROWTH)) {
                #pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 2));
                    if (top[r] > m[r]) {
                        const float f = factor_of((m[r] - top[r]) * c);
                        m[r] = top[r];
                        l[r] *= f;
                        #pragma unroll
                        for (int t = 0; t < NK * 2; ++t) { o[t][2 * r] *= f; o[t][2 * r + 1] *= f; }
                    }
                }
            }
            uint32_t hi[4], rest[4];
            #pragma unroll
            for (int r = 0; r < 2; ++r) {                                // row lane / 4 + 8 r
                const float off = SHIFT - (m[r] == -INFINITY ? 0.f : m[r] * c);
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float w0 = exp2_fast(fmaf(s[e][2 * r], c, off)), w1 = exp2_fast(fmaf(s[e][2 * r + 1], c, off));
                    l[r] += w0 + w1;
                    // the weights as two numbers of the values' type, so that their rounding does not reach the result
                    hi[2 * e + r] = Mma<E>::pack(w0, w1);
                    const float2 back = Mma<E>::unpack(hi[2 * e + r]);
                    rest[2 * e + r] = Mma<E>::pack(w0 - back.x, w1 - back.y);
                }
            }
            if constexpr (!APART) {
                #pragma unroll
                for (int t = 0; t < NK; ++t) {
                    uint32_t f[4];
                    const int row = (lane & 7) + 8 * ((lane >> 3) & 1), pc = (t & 3) * 2 + (lane >> 4);
                    ldsm4t(f, vt + (t >> 2) * (GROUP * 128) + row * 128 + ((pc ^ (row & 7)) * 16));
                    Mma<E>::run(o[2 * t], hi, f[0], f[1]);
                    Mma<E>::run(o[2 * t], rest, f[0], f[1]);
                    Mma<E>::run(o[2 * t + 1], hi, f[2], f[3]);
                    Mma<E>::run(o[2 * t + 1], rest, f[2], f[3]);
                }
            } else {
                const uint32_t one[4] = {Mma<E>::ONES, Mma<E>::ONES, Mma<E>::ONES, Mma<E>::ONES};
                #pragma unroll
                for (int t = 0; t < NK; ++t) {
                    uint32_t f[4], g[4];
                    const int row = (lane & 7) + 8 * ((lane >> 3) & 1), pc = (t & 3) * 2 + (lane >> 4);
                    ldsm4t(f, vt + (t >> 2) * (GROUP * 128) + row * 128 + ((pc ^ (row & 7)) * 16));
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        constexpr uint32_t INF = Mma<E>::INF;
                        g[e] = f[e] & (((f[e] & INF) == INF ? 0x0000FFFFu : 0u) | ((f[e] & (INF << 16)) == INF << 16 ? 0xFFFF0000u : 0u));
                        f[e] ^= g[e];
                    }
                    #pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        Mma<E>::run(o[2 * t + e], hi, f[2 * e], f[2 * e + 1]);
                        Mma<E>::run(o[2 * t + e], rest, f[2 * e], f[2 * e + 1]);
                        Mma<E>::run(o[2 * t + e], one, g[2 * e], g[2 * e + 1]);
                    }
                }
            }
            __syncwarp();                                                // every lane has read the stage
            if (lane == 0 && x + STAGES * stride < x1) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                load(x + STAGES * stride, stage);
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
    };
    walk(std::false_type());
    {
        float nan[4] = {o[0][0], o[0][1], o[0][2], o[0][3]};
        #pragma unroll
        for (int t = 1; t < NK * 2; ++t)
            #pragma unroll
            for (int f = 0; f < 4; f += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(nan[(t & 1) * 2 + f / 2]) : "f"(o[t][f]), "f"(o[t][f + 1]));
        asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(nan[0]) : "f"(nan[1]), "f"(nan[2]));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(nan[0]) : "f"(nan[3]));
        if (__builtin_expect(__any_sync(0xFFFFFFFFu, nan[0] != nan[0]) && ok, 0)) {             // once more: twice the time of a group that holds one
            if (lane == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            load_first();
            walk(std::true_type());
        }
    }
    #pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
    }

    // a row's value: the output, or its part
    const auto put = [&](uint32_t row, uint32_t d, float top, float weight, float sum) {
        if (a.parts > 0) {
            const int64_t at = ((int64_t)b * a.L + i) * a.H + h0 + row;
            part_sum(a, at, a.part0)[d] = sum;
            if (d == 0) *part_weight(a, at, a.part0) = make_float2(top, weight);
        } else {
            Mma<E>::store(a.out, (int64_t)b * a.os[0] + (int64_t)i * a.os[1] + (int64_t)(h0 + row) * a.os[2] + d, weight == 0.f ? 0.f : sum / weight);
        }
    };
    float* block = reinterpret_cast<float*>(smem + Sh::JOIN);
    float* block_w = block + 16 * Sh::DP;

    // join the warps: [warp][16][DP] sums, then [warp][16] maxima and weights
    __syncthreads();
    float* js = reinterpret_cast<float*>(smem);
    float* jm = js + RW * 16 * Sh::DP;
    #pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = lane / 4 + 8 * r;
        #pragma unroll
        for (int t = 0; t < NK * 2; ++t)
            *reinterpret_cast<float2*>(js + (warp * 16 + row) * Sh::DP + t * 8 + (lane & 3) * 2) = make_float2(o[t][2 * r], o[t][2 * r + 1]);
        if ((lane & 3) == 0) {                                       // (weights are 2^(x c - m c + SHIFT))
            jm[(warp * 16 + row) * 2] = m[r] == -INFINITY ? m[r] : m[r] * c - SHIFT;
            jm[(warp * 16 + row) * 2 + 1] = l[r];
        }
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < rows * a.D; x += RW * 32) {
        const uint32_t row = x / a.D, d = x - row * a.D;
        float top = -INFINITY, sum = 0.f, weight = 0.f;
        #pragma unroll
        for (int w = 0; w < RW; ++w) top = fmaxf(top, jm[(w * 16 + row) * 2]);
        const float ref = top == -INFINITY ? 0.f : top;
        #pragma unroll
        for (int w = 0; w < RW; ++w) {
            const float f = factor_of(jm[(w * 16 + row) * 2] - ref);
            sum = fmaf(js[(w * 16 + row) * Sh::DP + d], f, sum);
            weight = fmaf(jm[(w * 16 + row) * 2 + 1], f, weight);
        }
        if (slot >= 0) {
            slot_sum(a, blockIdx.x, slot, row)[d] = sum;
            if (d == 0) *slot_weight(a, blockIdx.x, slot, row) = make_float2(top, weight);
        } else if (!a.shared && a.cluster > 1) {
            block[row * Sh::DP + d] = sum;
            if (d == 0) { block_w[row * 2] = top; block_w[row * 2 + 1] = weight; }
        } else put(row, d, top, weight, sum);
    }
    if (!a.shared && a.cluster > 1) {
        // the cluster's parts: every block takes its share of the outputs and reads all blocks' values of them
        cluster_meet();
        for (uint32_t x = rank * RW * 32 + threadIdx.x; x < rows * a.D; x += a.cluster * RW * 32) {
            const uint32_t row = x / a.D, d = x - row * a.D, at = smem_u32(block + row * Sh::DP + d), wat = smem_u32(block_w + row * 2);
            float tops[8], weights[8], sums[8], top = -INFINITY, sum = 0.f, weight = 0.f;
            #pragma unroll
            for (int k = 0; k < 8; ++k) {
                tops[k] = -INFINITY; weights[k] = sums[k] = 0.f;
                if (k < a.cluster) { tops[k] = peer_load(wat, k); weights[k] = peer_load(wat + 4, k); sums[k] = peer_load(at, k); }
            }
            #pragma unroll
            for (int k = 0; k < 8; ++k) if (weights[k] != 0.f) top = fmaxf(top, tops[k]);
            const float ref = top == -INFINITY ? 0.f : top;
            #pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (weights[k] == 0.f) continue;                     // (a NaN is no zero)
                const float f = factor_of(tops[k] - ref);
                sum = fmaf(sums[k], f, sum);
                weight = fmaf(weights[k], f, weight);
            }
            put(row, d, top, weight, sum);
        }
        cluster_meet();                                              // (the others still read this block's memory)
    }
    w0 += take;
    if (a.shared && w0 < w1) {
        if (w0 >= table[token + 1] * groups) ++token;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();                                             // the join's memory becomes the ring again
    }
    }
    __syncthreads();
    if (*abort_flag) {
        // let copies that may still be in flight land before the block's shared memory is released
        const unsigned long long t0 = gtime_ns();
        while (gtime_ns() - t0 < 200000ull) { }
        __syncthreads();
    }
    end_beside(a);
}

// W warps join a row's parts: the tensor-core kernel's, and the few-row kernel's part or slots.  Maxima, then weights and
// sums relative to the largest.  A chain of dependent loads, bound by their latency: the blocks of a group come from its
// table entry, and with few rows four warps share a row's parts (8 rows of 37 parts: 8.4 -> 5 us).
template <class E, int W>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ AttnArgs a, uint32_t tiles)
{
    __shared__ float sums[W > 1 ? W : 1][128], weights[W > 1 ? W : 1];
    grid_dependency_wait();
    dependents_may_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = W > 1 ? warp : 0;
    const uint32_t row = W > 1 ? blockIdx.x : blockIdx.x * 4 + warp;
    if (row >= a.B * a.L * a.H) return;
    const uint32_t token = row / a.H, h = row - token * a.H;
    int first = 0, count = a.parts, listed = a.parts, gr = 0;       // parts 0 .. listed - 1 lie in the row's list, the rest in slots
    if (a.shared) {
        const uint32_t hk = h / a.G, gg = h - hk * a.G;
        gr = (int)(gg & 15);
        const int2 blocks = behind_wait(a.table)[(int64_t)token * (a.Hkv * tiles) + hk * tiles + gg / 16];
        first = blocks.x;
        if (blocks.y > 0) {
            if (listed > 0) --listed;                                // (the entry for an undivided group is not in use)
            count = listed + blocks.y;
        } else if (a.parts == 0) return;                             // undivided: written already
    }
    const auto weight_of = [&](int s) { return s < listed ? *part_weight(a, row, s) : *slot_weight(a, first + s - listed, s == listed, gr); };
    const auto sum_of = [&](int s) { return (s < listed ? part_sum(a, row, s) : slot_sum(a, first + s - listed, s == listed, gr)); };
    float top = -INFINITY;
    for (int s = lane; s < count; s += 32) {
        const float2 ml = weight_of(s);
        if (ml.y != 0.f) top = fmaxf(top, ml.x);
    }
    #pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
    const float ref = top == -INFINITY ? 0.f : top;
    float weight = 0.f, sum[4] = {};
    const bool in = lane * 4 < (int)a.D;
    for (int s0 = sub; s0 < count; s0 += 32 * W) {                   // this warp's parts: s0, s0 + W, ...
        float f = 0.f;
        if (s0 + lane * W < count) {
            const float2 ml = weight_of(s0 + lane * W);
            if (ml.y != 0.f) { f = factor_of(ml.x - ref); weight = fmaf(ml.y, f, weight); }
        }
        const int end = min(32, (count - s0 + W - 1) / W);
        #pragma unroll 8
        for (int s = 0; s < end; ++s) {
            const float g = __shfl_sync(0xFFFFFFFFu, f, s);
            if (g != 0.f && in) {                                    // an empty part's sums are not looked at (a NaN is no zero)
                const float4 x = *reinterpret_cast<const float4*>(sum_of(s0 + s * W) + lane * 4);
                sum[0] = fmaf(x.x, g, sum[0]); sum[1] = fmaf(x.y, g, sum[1]); sum[2] = fmaf(x.z, g, sum[2]); sum[3] = fmaf(x.w, g, sum[3]);
            }
        }
    }
    #pragma unroll
    for (int k = 16; k; k >>= 1) weight += __shfl_xor_sync(0xFFFFFFFFu, weight, k);
    if (W > 1) {
        #pragma unroll
        for (int e = 0; e < 4; ++e) sums[sub][lane * 4 + e] = sum[e];
        if (lane == 0) weights[sub] = weight;
        __syncthreads();
        if (warp > 0) return;
        #pragma unroll
        for (int w = 1; w < W; ++w) {
            weight += weights[w];
            #pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += sums[w][lane * 4 + e];
        }
    }
    const uint32_t b = token / a.L, i = token - b * a.L;
    if (in) {
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            Mma<E>::store(a.out, (int64_t)b * a.os[0] + (int64_t)i * a.os[1] + (int64_t)h * a.os[2] + lane * 4 + e, weight == 0.f ? 0.f : sum[e] / weight);
    }
}

template <class E>
int join_launch(const AttnArgs& a, cudaStream_t stream)
{
    const int64_t rows = (int64_t)a.B * a.L * a.H;
    if (rows > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    const uint32_t tiles = (a.G + 15) / 16;
    // (64 x 32 rows: four warps a row 81 us, one 88, of the whole call; 33536 rows: 175 and 152)
    if (rows <= 4096) HBQ_CUDA_TRY(launch_dependent(attention_join_kernel<E, 4>, (unsigned)rows, 128, 0, stream, a, tiles));
    else HBQ_CUDA_TRY(launch_dependent(attention_join_kernel<E, 1>, (unsigned)((rows + 3) / 4), 128, 0, stream, a, tiles));
    HBQ_LAUNCH_CHECK("attention_join_kernel");
    return HBQ_OK;
}

template <class E, int NK>
int rows_launch(const AttnArgs& a, const RowsMaps& maps, cudaStream_t stream)
{
    { const int rc = ensure_dynamic_smem(attention_rows_kernel<E, NK>, RowsShape<NK>::BYTES); if (rc) return rc; }
    const unsigned cluster = a.shared ? 1u : (unsigned)a.cluster;
    HBQ_CUDA_TRY(launch_dependent_clusters(attention_rows_kernel<E, NK>, (unsigned)a.blocks, cluster, RW * 32, (size_t)RowsShape<NK>::BYTES, stream, a, maps, (a.G + 15) / 16));
    HBQ_LAUNCH_CHECK("attention_rows_kernel");
    return HBQ_OK;
}

template <class E>
int rows_type(const AttnArgs& a, const RowsMaps& maps, cudaStream_t stream)
{
    switch ((a.D + 15) / 16) {
        case 1: case 2: case 3: case 4: return rows_launch<E, 4>(a, maps, stream);
        case 5: return rows_launch<E, 5>(a, maps, stream);
        case 6: return rows_launch<E, 6>(a, maps, stream);
        case 7: return rows_launch<E, 7>(a, maps, stream);
        default: return rows_launch<E, 8>(a, maps, stream);
    }
}

}  // namespace

// Blocks of the few-row kernel; prefix: a row's list begins with it.  A cluster of up to eight blocks a row group as far as
// all are resident at once and none has more than 512 keys (8 steps a warp); else shares of equal size over the blocks that are
// resident, or a block a group where there are too many tokens for the table.  us, 32 / 8 heads of 128, clusters and shares:
// one sequence of 512 keys 8.9 and 9.2, 4096 12.2 and 16.7, 8192 18 and 19, 16384 30 and 22; 8 of 2048 14.9 and 22; 64 of 512
// (a block each) 31 and 37.  256 sequences in shares and 257 in blocks: 1024 keys each 169 and 177, 16 to 1024 of them 130 and 106, one of
// 32768 among 512s 117 and 427.  `*small`: all row groups are resident and have no more keys than that.
int attention_rows_blocks(const hbq_attention* p, bool prefix, int* shared, int* cluster, bool* small)
{
    int sms = 148;
    device_sms(&sms);
    const int64_t all = p->Hkv * ((p->H / p->Hkv + 15) / 16) * p->B * p->L, most = BLOCKS_PER_SM * sms;
    int64_t keys = p->S;
    if (p->window > 0 && p->window + p->sinks < keys) keys = p->window + p->sinks;
    if (prefix) keys += p->P;
    int c = 8;
    while (c > 1 && (all * c > most || keys <= 64 * (c / 2))) c /= 2;
    *small = all <= most && keys <= 512 * c;
    *shared = keys > 512 * c && p->B * p->L <= RW * 64;
    *cluster = *shared || keys > 512 * c ? 1 : c;
    if (!*shared) return all > 0x7FFFFFFF / 8 ? -1 : (int)(all * *cluster);
    const int64_t units = ((keys + RW * GROUP - 1) / (RW * GROUP) + 1) * all;
    return (int)(units < most ? units : most);
}

int attention_rows_launch(const AttnArgs& a, int dtype, cudaStream_t stream)
{
    RowsMaps maps = {};
    int rc = HBQ_OK;
    if (a.S > 0) {
        rc = attention_cache_map(&maps.k, a.k, dtype, a.D, GROUP, a.S, a.ks[2], a.Hkv, a.ks[1], a.B, a.ks[0]);
        if (!rc) rc = attention_cache_map(&maps.v, a.v, dtype, a.D, GROUP, a.S, a.vs[2], a.Hkv, a.vs[1], a.B, a.vs[0]);
    }
    if (a.P > 0 && !rc) {
        rc = attention_cache_map(&maps.pk, a.pk, dtype, a.D, GROUP, a.P, a.pks[1], a.Hkv, a.pks[0], 1, 0);
        if (!rc) rc = attention_cache_map(&maps.pv, a.pv, dtype, a.D, GROUP, a.P, a.pvs[1], a.Hkv, a.pvs[0], 1, 0);
    }
    if (rc) return rc;
    return dtype == HBQ_DTYPE_F16 ? rows_type<__half>(a, maps, stream) : rows_type<__nv_bfloat16>(a, maps, stream);
}

int attention_rows_status(int* host_out)
{
    HBQ_CUDA_TRY(cudaMemcpyFromSymbol(host_out, g_tc_status, sizeof(int)));
    return HBQ_OK;
}
int attention_rows_status_reset()
{
    const int z = 0;
    HBQ_CUDA_TRY(cudaMemcpyToSymbol(g_tc_status, &z, sizeof(int)));
    return HBQ_OK;
}

int attention_join_launch(const AttnArgs& a, int dtype, cudaStream_t stream)
{
    return dtype == HBQ_DTYPE_F16 ? join_launch<__half>(a, stream) : join_launch<__nv_bfloat16>(a, stream);
}

}  // namespace hbq
