// Rotary positions of projected heads, with 64-bit angles, after an RMS norm of every head where there is one.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (norm only)
//   (u, v) -> factor * (u cos a - v sin a, v cos a + u sin a),   a = position * inv_freq[i], for each pair i
//
// Bound by memory: each value is read once and written once.  A position's angles are the same for all of its heads, so a
// block computes them once into shared memory: the product and its reduction to a part of a turn in 64 bits (at position
// 10^6 an angle in 32 bits is off by 0.06), cosine and sine of that part in 32 bits.  A table of them would be read
// from memory in their place and has to be kept for every position.
#include "common.cuh"

namespace hbq {

namespace {

struct HeadsArg {
    const void* data;
    void* out;
    const void* weight;
    int64_t sb, st, sh, ob, ot, oh;
};
struct RotaryArgs {
    HeadsArg x[2];                 // queries and keys; the second is empty for one tensor
    const double* inv_freq;
    const void* positions;
    int64_t pb, pt, tokens;        // tokens = B * T
    uint32_t T, heads0, heads, D, rot, groups;
    int interleaved, positions_64;
    float factor, eps;
    int tokens_per_block;
};

constexpr int WARPS = 8;

template <class E> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(bits_h2(u)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) { return h2_bits(__floats2half2_rn(a, b)); }
    static __device__ __forceinline__ float up1(const void* p, int64_t i) { return __half2float(static_cast<const __half*>(p)[i]); }
    static __device__ __forceinline__ void down1(void* p, int64_t i, float v) { static_cast<__half*>(p)[i] = __float2half_rn(v); }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 up(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t down(float a, float b)
    {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float up1(const void* p, int64_t i) { return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]); }
    static __device__ __forceinline__ void down1(void* p, int64_t i, float v) { static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); }
};

// Cosine and sine of position * inv_freq: in turns, so that the reduction is a subtraction of the nearest whole number.
__device__ __forceinline__ float2 turn(int64_t position, double inv_freq, float factor)
{
    const double t = (double)position * (inv_freq * 0.15915494309189535);       // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    return make_float2(c * factor, s * factor);
}
__device__ __forceinline__ void rotate(float& u, float& v, float2 cs)
{
    const float r = fmaf(u, cs.x, -(v * cs.y));
    v = fmaf(v, cs.x, u * cs.y);
    u = r;
}
__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t token)
{
    const int64_t b = token / a.T, t = token - b * a.T, i = b * a.pb + t * a.pt;
    return a.positions_64 ? static_cast<const int64_t*>(a.positions)[i] : static_cast<const int32_t*>(a.positions)[i];
}

// Heads whose length and turning part are multiples of 16: a lane holds two runs of 8 values, which the rotation pairs
// with one another (runs c and c + rot / 16 of the half layout, neighbours of the interleaved one), so that a pair never
// leaves its lane; LANES lanes share a head and 32 / LANES heads a warp.  Each lane needs the 8 angles from 8 c on.
// A block takes `tokens_per_block` tokens: eight where there are many, so that a warp keeps one token's angles in
// registers over all its heads; one where there are few, its heads spread over the warps and over blockIdx.y.
template <class E, int LANES, bool NORM>
__global__ void __launch_bounds__(WARPS * 32) rotary_kernel(const __grid_constant__ RotaryArgs a)
{
    extern __shared__ float2 angles[];             // [tokens_per_block][rot / 2]
    grid_dependency_wait();
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & (LANES - 1), sub = lane / LANES;
    const uint32_t half = a.rot / 2, tpb = (uint32_t)a.tokens_per_block;
    const int64_t token0 = (int64_t)blockIdx.x * tpb;
    const uint32_t here = (uint32_t)min((int64_t)tpb, a.tokens - token0);
    const double* freq = behind_wait(a.inv_freq);
    for (uint32_t i = threadIdx.x; i < here * half; i += WARPS * 32) {
        const uint32_t t = i / half;
        angles[i] = turn(position_of(a, token0 + t), freq[i - t * half], a.factor);
    }
    __syncthreads();

    const bool in_head = (uint32_t)c * 16 < a.D, turns = (uint32_t)c * 16 < a.rot;
    uint32_t d0, d1;                               // where the lane's two runs begin
    if (a.interleaved || !turns) { d0 = 16 * c; d1 = d0 + 8; }
    else { d0 = 8 * c; d1 = d0 + half; }
    float w[2][16];
    if (NORM) {
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
            const void* wp = a.x[j].weight;
            #pragma unroll
            for (int r = 0; r < 2; ++r) {
                uint4 u = make_uint4(0, 0, 0, 0);
                if (in_head && wp) u = *reinterpret_cast<const uint4*>(static_cast<const E*>(wp) + (r ? d1 : d0));
                const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
                #pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float2 f = Pair<E>::up(ww[p]);
                    w[j][8 * r + 2 * p] = f.x; w[j][8 * r + 2 * p + 1] = f.y;
                }
            }
        }
    }
    float2 cs[8];
    uint32_t cur = 0xFFFFFFFFu;
    int64_t b = 0, t = 0;
    constexpr uint32_t PER = 32 / LANES;
    const uint32_t items = here * a.groups, stride = WARPS * gridDim.y;
    for (uint32_t it = blockIdx.y * WARPS + warp; it < items; it += stride) {
        // (tokens of a block innermost: with eight of them a warp keeps its own)
        const uint32_t g = it / here, tk = it - g * here;
        if (tk != cur) {
            cur = tk;
            b = (token0 + tk) / a.T; t = token0 + tk - b * a.T;
            if (turns) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) cs[i] = angles[tk * half + 8 * c + i];
            }
        }
        const uint32_t h = g * PER + sub;
        const bool second = h >= a.heads0, live = h < a.heads && in_head;
        const HeadsArg& x = a.x[second ? 1 : 0];
        const int64_t hh = second ? h - a.heads0 : h;
        uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
        if (live) {
            const E* p = static_cast<const E*>(x.data) + b * x.sb + t * x.st + hh * x.sh;
            u0 = *reinterpret_cast<const uint4*>(p + d0);
            u1 = *reinterpret_cast<const uint4*>(p + d1);
        }
        float v[16];
        {
            const uint32_t uu[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
            #pragma unroll
            for (int p = 0; p < 8; ++p) {
                const float2 f = Pair<E>::up(uu[p]);
                v[2 * p] = f.x; v[2 * p + 1] = f.y;
            }
        }
        if (NORM) {
            float s = 0.f;
            #pragma unroll
            for (int i = 0; i < 16; ++i) s = fmaf(v[i], v[i], s);
            #pragma unroll
            for (int m = LANES / 2; m; m >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, m);
            s = rsqrtf(s / (float)a.D + a.eps);
            #pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= s * (second ? w[1][i] : w[0][i]);
        }
        if (turns) {
            if (a.interleaved) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) rotate(v[2 * i], v[2 * i + 1], cs[i]);
            } else {
                #pragma unroll
                for (int i = 0; i < 8; ++i) rotate(v[i], v[8 + i], cs[i]);
            }
        }
        if (live) {
            E* o = static_cast<E*>(x.out) + b * x.ob + t * x.ot + hh * x.oh;
            *reinterpret_cast<uint4*>(o + d0) = make_uint4(Pair<E>::down(v[0], v[1]), Pair<E>::down(v[2], v[3]), Pair<E>::down(v[4], v[5]), Pair<E>::down(v[6], v[7]));
            *reinterpret_cast<uint4*>(o + d1) = make_uint4(Pair<E>::down(v[8], v[9]), Pair<E>::down(v[10], v[11]), Pair<E>::down(v[12], v[13]), Pair<E>::down(v[14], v[15]));
        }
    }
}

// Every other head length, turning part, stride and alignment: a warp per head, value by value.  A lane reads both values
// of a pair before it writes either, and the norm's sum is complete before any is written, so `out` may be the input.
template <class E, bool NORM>
__global__ void __launch_bounds__(WARPS * 32) rotary_any_kernel(const __grid_constant__ RotaryArgs a)
{
    grid_dependency_wait();
    dependents_may_start();
    const double* freq = behind_wait(a.inv_freq);
    const uint32_t lane = threadIdx.x & 31, half = a.rot / 2;
    const int64_t total = a.tokens * a.heads;
    for (int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * WARPS) {
        const int64_t token = i / a.heads, b = token / a.T, t = token - b * a.T;
        uint32_t h = (uint32_t)(i - token * a.heads);
        const bool second = h >= a.heads0;
        const HeadsArg& x = a.x[second ? 1 : 0];
        if (second) h -= a.heads0;
        const int64_t in = b * x.sb + t * x.st + h * x.sh, on = b * x.ob + t * x.ot + h * x.oh;
        float s = 1.f;
        if (NORM) {
            s = 0.f;
            for (uint32_t d = lane; d < a.D; d += 32) { const float v = Pair<E>::up1(x.data, in + d); s = fmaf(v, v, s); }
            #pragma unroll
            for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, m);
            s = rsqrtf(s / (float)a.D + a.eps);
        }
        const int64_t position = position_of(a, token);
        for (uint32_t p = lane; p < half; p += 32) {
            const uint32_t d0 = a.interleaved ? 2 * p : p, d1 = a.interleaved ? d0 + 1 : p + half;
            float u = Pair<E>::up1(x.data, in + d0), v = Pair<E>::up1(x.data, in + d1);
            if (NORM) { u *= s * Pair<E>::up1(x.weight, d0); v *= s * Pair<E>::up1(x.weight, d1); }
            const float2 cs = turn(position, freq[p], a.factor);
            rotate(u, v, cs);
            Pair<E>::down1(x.out, on + d0, u);
            Pair<E>::down1(x.out, on + d1, v);
        }
        for (uint32_t d = a.rot + lane; d < a.D; d += 32) {
            float v = Pair<E>::up1(x.data, in + d);
            if (NORM) v *= s * Pair<E>::up1(x.weight, d);
            Pair<E>::down1(x.out, on + d, v);
        }
    }
}

template <class E, int LANES, bool NORM>
int launch_lanes(RotaryArgs& a, int sms, cudaStream_t stream)
{
    constexpr int PER = 32 / LANES;
    a.groups = (a.heads + PER - 1) / PER;
    a.tokens_per_block = a.tokens >= (int64_t)sms * 16 ? 8 : 1;
    const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    if (blocks > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    const unsigned split = a.tokens_per_block > 1 ? 1u : (a.groups + WARPS - 1) / WARPS;
    HBQ_CUDA_TRY(launch_dependent(rotary_kernel<E, LANES, NORM>, dim3((unsigned)blocks, split), WARPS * 32,
                                  (size_t)a.tokens_per_block * (a.rot / 2) * sizeof(float2), stream, a));
    HBQ_LAUNCH_CHECK("rotary_kernel");
    return HBQ_OK;
}

template <class E, bool NORM>
int launch_type(RotaryArgs& a, bool runs, cudaStream_t stream)
{
    int sms = 0;
    { const int rc = device_sms(&sms); if (rc) return rc; }
    if (runs) {
        const uint32_t lanes = a.D / 16;
        if (lanes <= 4) return launch_lanes<E, 4, NORM>(a, sms, stream);
        if (lanes <= 8) return launch_lanes<E, 8, NORM>(a, sms, stream);
        return launch_lanes<E, 16, NORM>(a, sms, stream);
    }
    const int64_t need = (a.tokens * a.heads + WARPS - 1) / WARPS, cap = (int64_t)sms * 8;
    HBQ_CUDA_TRY(launch_dependent(rotary_any_kernel<E, NORM>, (unsigned)(need < cap ? need : cap), WARPS * 32, 0, stream, a));
    HBQ_LAUNCH_CHECK("rotary_any_kernel");
    return HBQ_OK;
}

// The vector kernel's terms for one tensor: 16-byte runs everywhere.
bool in_runs(const hbq_heads* x)
{
    int64_t s = 0;
    for (int i = 0; i < 3; ++i) s |= x->stride[i] | x->out_stride[i];
    return (s % 8) == 0 && ((reinterpret_cast<uintptr_t>(x->data) | reinterpret_cast<uintptr_t>(x->out) | reinterpret_cast<uintptr_t>(x->weight)) & 15) == 0;
}

}  // namespace

int rotary_launch(const hbq_heads* q, const hbq_heads* k, const hbq_rotary* r, int dtype, int64_t B, int64_t T, int64_t D,
                  bool norm, float eps, cudaStream_t stream)
{
    if (!q || !r || B < 0 || T < 0 || D <= 0 || q->heads < 0 || (k && k->heads < 0)) return HBQ_ERR_ARG;
    if (dtype != HBQ_DTYPE_F16 && dtype != HBQ_DTYPE_BF16) return HBQ_ERR_ARG;
    if (r->rot < 2 || (r->rot & 1) || r->rot > D) return HBQ_ERR_ARG;
    const int64_t heads = q->heads + (k ? k->heads : 0);
    if (B == 0 || T == 0 || heads == 0) return HBQ_OK;
    if (!r->inv_freq || !r->positions) return HBQ_ERR_ARG;
    if (D > (1 << 20) || heads > (1 << 20) || T > 0x7FFFFFFFll || B > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    RotaryArgs a = {};
    const hbq_heads* x[2] = {q, k};
    bool runs = (D % 16) == 0 && D <= 256 && (r->rot % 16) == 0;
    for (int i = 0; i < 2; ++i) {
        if (!x[i] || x[i]->heads == 0) continue;
        if (!x[i]->data || !x[i]->out || (norm && !x[i]->weight)) return HBQ_ERR_ARG;
        a.x[i] = {x[i]->data, x[i]->out, x[i]->weight, x[i]->stride[0], x[i]->stride[1], x[i]->stride[2],
                  x[i]->out_stride[0], x[i]->out_stride[1], x[i]->out_stride[2]};
        runs = runs && in_runs(x[i]);
    }
    a.inv_freq = r->inv_freq; a.positions = r->positions; a.pb = r->pos_stride[0]; a.pt = r->pos_stride[1];
    a.tokens = B * T; a.T = (uint32_t)T; a.heads0 = (uint32_t)q->heads; a.heads = (uint32_t)heads;
    a.D = (uint32_t)D; a.rot = (uint32_t)r->rot; a.interleaved = r->interleaved != 0; a.positions_64 = r->positions_64 != 0;
    a.factor = r->factor; a.eps = eps;
    if (dtype == HBQ_DTYPE_F16) return norm ? launch_type<__half, true>(a, runs, stream) : launch_type<__half, false>(a, runs, stream);
    return norm ? launch_type<__nv_bfloat16, true>(a, runs, stream) : launch_type<__nv_bfloat16, false>(a, runs, stream);
}

}  // namespace hbq
