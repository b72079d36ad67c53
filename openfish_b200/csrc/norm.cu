// norm.cu -- residual, norm and 8-bit tokens, row by row (openfish_b200_norm).
//
//   s = x + alpha r;  y = (s - mean) / sqrt(var + eps) w + b  (or without the mean, or y = s);  out = y in 16 bits;
//   q = round(127 y / max|y|), scale = max|y| / 127
//
// One pass over memory: a row's s stays in the registers of the warp or block that read it, so the mean, the
// variance about that mean (two sums, no cancellation), the largest |y| and the results all come from there.  What
// bounds it is HBM: 2 bytes for each of x, r, out and 1 for q.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "encoder.h"
#include "encoder_device.cuh"

namespace {

using ofe::add2;
using ofe::fma2;
using ofe::from_float;
using ofe::mul2;
using ofe::to_float;

template <class T>
struct NormArgs {
    const T *x, *r, *w, *b;
    T *out;
    int8_t *q;
    float *q_scale;
    long long x_stride, r_stride, out_stride, q_stride, rows;
    int width, kind;
    float eps, alpha;
    bool w_packs, q_packs;  // weight and bias, the codes' rows: on boundaries of a pack, whatever the rows of x are on
};

// V elements that lie together, two at a time: 16 bytes where everything is aligned to that, else one element (and a
// zero beside it).
template <class T, int V>
__device__ __forceinline__ void read(const T *p, float2 (&f)[(V + 1) / 2]) {
    if (V == 8) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        f[0] = ofe::unpack<T>(w.x);
        f[V / 8] = ofe::unpack<T>(w.y);
        f[V / 4] = ofe::unpack<T>(w.z);
        f[V / 8 * 3] = ofe::unpack<T>(w.w);
    } else {
        f[0] = make_float2(to_float(*p), 0.f);
    }
}
template <class T, int V>
__device__ __forceinline__ void write(T *p, const float2 (&f)[(V + 1) / 2]) {
    if (V == 8)
        *reinterpret_cast<uint4 *>(p) = make_uint4(ofe::pack<T>(f[0].x, f[0].y), ofe::pack<T>(f[V / 8].x, f[V / 8].y),
                                                   ofe::pack<T>(f[V / 4].x, f[V / 4].y), ofe::pack<T>(f[V / 8 * 3].x, f[V / 8 * 3].y));
    else
        *p = from_float<T>(f[0].x);
}

// A sum (or maximum) over the threads of a row: its warp, or all warps of the block through shared memory.
template <bool BLOCK, class Op>
__device__ __forceinline__ float reduce(float v, float *scratch, Op op) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
    if (BLOCK) {
        const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
        __syncthreads();  // the last reduction's readers are done
        if (lane == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        v = scratch[lane < warps ? lane : 0];
        // every warp adds the same numbers in the same order; lanes beyond the last warp hold the neutral element
        if (lane >= warps) v = op(0.f, 0.f);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
    }
    return v;
}

// BLOCK: a block to a row, else a warp.  CH packs of V elements to a thread.
// SHIFT: rows that start anywhere, all tensors' in the same place between two 16-byte boundaries.  The packs are the aligned 16 bytes
// around the row, and which thread has which element does not matter to a sum: elements of a pack that lie in front of the row or
// behind it are taken as zeros and not written.
template <class T, int V, int CH, bool BLOCK, bool SHIFT>
__global__ void __launch_bounds__(BLOCK ? 1024 : 128) norm_kernel(const NormArgs<T> a) {
    __shared__ float scratch[32];
    __shared__ uint64_t firsts[BLOCK && SHIFT ? CH : 1][32];  // the codes of each warp's first thread
    constexpr int P = (V + 1) / 2;
    const int lane = BLOCK ? threadIdx.x : threadIdx.x & 31;
    const int lanes = BLOCK ? blockDim.x : 32;
    const long long step = BLOCK ? gridDim.x : (long long)gridDim.x * (blockDim.x >> 5);
    const long long first = BLOCK ? blockIdx.x : (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const auto add = [](float p, float q) { return p + q; };
    const auto most = [](float p, float q) { return fmaxf(p, q); };
    const float inv = 1.f / (float)a.width;

    for (long long row = first; row < a.rows; row += step) {
        const T *const x = a.x + row * a.x_stride, *const r = a.r + row * a.r_stride;
        const int shift = SHIFT ? (int)((uintptr_t)x & 15) / 2 : 0;
        const auto place = [&](int c) { return (c * lanes + lane) * V - shift; };            // a pack's first element
        const auto here = [&](int at) { return at < a.width && (!SHIFT || at > -V); };        // whether it has any of the row
        const auto whole = [&](int at) { return !SHIFT || (at >= 0 && at + V <= a.width); };  // or nothing else
        const auto trim = [&](int at, float2 (&f)[P]) {  // nothing but the row's elements
            if (whole(at)) return;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (at + 2 * i < 0 || at + 2 * i >= a.width) f[i].x = 0.f;
                if (at + 2 * i + 1 < 0 || at + 2 * i + 1 >= a.width) f[i].y = 0.f;
            }
        };
        const auto along = [&](const T *p, int at, float2 (&f)[P]) {  // a weight or bias
            if (!SHIFT) {
                read<T, V>(p + at, f);
            } else if (a.w_packs) {
                // the two packs that the eight lie in, moved by n elements (the same n in the whole row)
                const int n = at & 7, k = at - n;
                uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
                if (k >= 0 && k < a.width) v0 = *reinterpret_cast<const uint4 *>(p + k);
                if (n > 0 && k + 8 < a.width) v1 = *reinterpret_cast<const uint4 *>(p + k + 8);
                uint32_t m[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int i = 0; i < 6; ++i) m[i] = n & 4 ? m[i + 2] : m[i];
#pragma unroll
                for (int i = 0; i < 5; ++i) m[i] = n & 2 ? m[i + 1] : m[i];
#pragma unroll
                for (int i = 0; i < P; ++i) f[i] = ofe::unpack<T>(n & 1 ? __byte_perm(m[i], m[i + 1], 0x5432) : m[i]);
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) f[i] = make_float2(to_float(p[min(max(at + 2 * i, 0), a.width - 1)]), to_float(p[min(max(at + 2 * i + 1, 0), a.width - 1)]));
            }
        };
        float2 s[CH][P];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = place(c);
#pragma unroll
            for (int i = 0; i < P; ++i) s[c][i] = {0.f, 0.f};
            if (here(at)) read<T, V>(x + at, s[c]);
        }
        if (a.r) {
            float2 f[CH][P];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int at = place(c);
                if (here(at)) {
                    read<T, V>(r + at, f[c]);
#pragma unroll
                    for (int i = 0; i < P; ++i) s[c][i] = fma2(f[c][i], {a.alpha, a.alpha}, s[c][i]);
                }
            }
        }
        if (SHIFT) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (here(place(c))) trim(place(c), s[c]);
        }
        if (a.kind != OPENFISH_B200_NORM_NONE) {
            float2 sum = {0.f, 0.f};
            if (a.kind == OPENFISH_B200_NORM_LAYER) {
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < P; ++i) sum = add2(sum, s[c][i]);
                const float mean = reduce<BLOCK>(sum.x + sum.y, scratch, add) * inv;
                sum = {0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int at = place(c);
                    if (here(at)) {
#pragma unroll
                        for (int i = 0; i < P; ++i) s[c][i] = add2(s[c][i], {-mean, V == 1 ? 0.f : -mean});
                        trim(at, s[c]);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < P; ++i) sum = fma2(s[c][i], s[c][i], sum);
            const float factor = 1.f / sqrtf(reduce<BLOCK>(sum.x + sum.y, scratch, add) * inv + a.eps);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int at = place(c);
                if (here(at)) {
                    float2 f[P];
#pragma unroll
                    for (int i = 0; i < P; ++i) s[c][i] = mul2(s[c][i], {factor, factor});
                    if (a.w) {
                        along(a.w, at, f);
#pragma unroll
                        for (int i = 0; i < P; ++i) s[c][i] = mul2(s[c][i], f[i]);
                    }
                    if (a.b) {
                        along(a.b, at, f);
#pragma unroll
                        for (int i = 0; i < P; ++i) s[c][i] = add2(s[c][i], f[i]);
                    }
                    trim(at, s[c]);
                }
            }
        }
        if (a.out) {
            T *const out = a.out + row * a.out_stride;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int at = place(c);
                if (!here(at)) continue;
                if (whole(at)) {
                    write<T, V>(out + at, s[c]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (at + i >= 0 && at + i < a.width) out[at + i] = from_float<T>(i & 1 ? s[c][i / 2].y : s[c][i / 2].x);
                }
            }
        }
        if (!a.q) continue;
        float top = 0.f;
        bool odd = false;  // an infinity or NaN in the row (a NaN is lost on a maximum; such a row counts as one with an infinity)
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                top = fmaxf(top, fmaxf(fabsf(s[c][i].x), fabsf(s[c][i].y)));
                odd |= !(fabsf(s[c][i].x) < INFINITY) | !(fabsf(s[c][i].y) < INFINITY);
            }
        top = reduce<BLOCK>(odd ? INFINITY : top, scratch, most);
        const bool fine = top < INFINITY;
        const float back = 127.f / top;  // no number for a row of zeros, and beyond fp32 for one whose top is below 2^-121
        const bool direct = back < INFINITY;
        int8_t *const q = a.q + row * a.q_stride;
        uint64_t codes[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            alignas(8) int8_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= V) break;
                const float y = i & 1 ? s[c][i / 2].y : s[c][i / 2].x;
                const float f = direct ? y * back : top > 0.f ? y / top * 127.f : 0.f;
                // (|f| is at most 127 and a rounding: no clamp can be reached)
                o[i] = fine ? (int8_t)__float2int_rn(f) : (int8_t)0;
            }
            if (V == 8) codes[c] = *reinterpret_cast<const uint64_t *>(o);
            else codes[c] = (uint8_t)o[0];
        }
        if (BLOCK && SHIFT && a.q_packs) {
            if ((lane & 31) == 0) {
#pragma unroll
                for (int c = 0; c < CH; ++c) firsts[BLOCK && SHIFT ? c : 0][lane >> 5] = codes[c];
            }
            __syncthreads();  // (what was there for the row before has been read: the largest |y| has been found since)
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = place(c);
            if (V == 8 && !SHIFT) {
                if (here(at)) *reinterpret_cast<uint64_t *>(q + at) = codes[c];
            } else if (V == 8 && a.q_packs) {
                // the eight codes from the next boundary on: the end of these and the beginning of the next thread's (behind the last
                // thread in a warp: the next warp's first one, or the first one's next pack)
                uint64_t after = __shfl_down_sync(0xffffffffu, codes[c], 1);
                const int to = at + shift;
                if (BLOCK) {
                    const int warp = lane >> 5;
                    if ((lane & 31) == 31) after = warp + 1 < lanes >> 5 ? firsts[SHIFT ? c : 0][warp + 1] : firsts[SHIFT && c + 1 < CH ? c + 1 : 0][0];
                } else if (CH > 1) {
                    const uint64_t first_next = __shfl_sync(0xffffffffu, codes[c + 1 < CH ? c + 1 : c], 0);
                    if (lane == 31) after = first_next;
                }
                const uint64_t both = shift == 0 ? codes[c] : codes[c] >> (8 * shift) | after << (64 - 8 * shift);
                if (to + 8 <= a.width) {
                    *reinterpret_cast<uint64_t *>(q + to) = both;
                } else {
                    for (int i = 0; to + i < a.width; ++i) q[to + i] = (int8_t)(both >> (8 * i));
                }
            } else if (here(at)) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (!SHIFT || (at + i >= 0 && at + i < a.width)) q[at + i] = (int8_t)(codes[c] >> (8 * i));
            }
        }
        if (lane == 0) a.q_scale[row] = fine ? top / 127.f : NAN;
    }
}

template <class T, int V, int CH, bool BLOCK, bool SHIFT>
void launch(const NormArgs<T> &a, int threads, int sms, cudaStream_t stream) {
    const long long per_block = BLOCK ? 1 : threads / 32;
    long long blocks = (a.rows + per_block - 1) / per_block;
    // Rows in turn for two blocks where one fits (53312 rows of 512 with a residual, us with one, two, four blocks: 32.2,
    // 31.1, 32.0; with a block to every four rows 32.8).
    const long long cap = (long long)sms * (2048 / threads) * 2;
    if (blocks > cap) blocks = cap;
    norm_kernel<T, V, CH, BLOCK, SHIFT><<<(unsigned)blocks, threads, 0, stream>>>(a);
}

// A warp to a row while 4 packs (of one element: 16) to a lane hold it, else a block with a few packs to a thread, so that an SM has several
// rows and as many packs on their way as its registers hold.  Layer norm with a residual, us: 30000 rows of 2048 with two packs to a thread 74,
// with one 88, and by warps with eight 88; 12000 of 4096 68, 83; 8000 of 8192 95, 130 (where rows start anywhere there is more to do for
// a pack, and one is better: 8000 of 5001 84, with two 90).  Beyond 8192, where one would take more than 1024 threads, four: 4000 of
// 9000 59, with four to each of 1024 threads 121; 2000 of 16000 56, 76.
// Single elements beyond 4096 (a result or residual whose rows start elsewhere than x's) take 32 to each of 1024 threads, more than its 32 registers: 2116
// bytes are stored and 2376 loaded again.  8000 of 5001, layer norm without a residual 1496, where all start alike 56.
template <class T, int V, bool SHIFT>
void dispatch(const NormArgs<T> &a, int sms, cudaStream_t stream) {
    const int packs = (a.width + V - 1) / V + SHIFT;
    constexpr int S = V == 8 ? 1 : 4;  // single elements are an eighth of a pack: more of them
    constexpr int B = V == 8 && !SHIFT ? 2 : S;
    if (packs <= 32 * S) launch<T, V, S, false, SHIFT>(a, 128, sms, stream);
    else if (packs <= 64 * S) launch<T, V, 2 * S, false, SHIFT>(a, 128, sms, stream);
    else if (packs <= 96 * S) launch<T, V, 3 * S, false, SHIFT>(a, 128, sms, stream);
    else if (packs <= 128 * S) launch<T, V, 4 * S, false, SHIFT>(a, 128, sms, stream);
    else if (packs <= 1024 * S) launch<T, V, B, true, SHIFT>(a, ((packs + B - 1) / B + 31) / 32 * 32, sms, stream);
    else if (V == 8 && packs <= 4096) launch<T, V, 4, true, SHIFT>(a, ((packs + 3) / 4 + 31) / 32 * 32, sms, stream);
    else launch<T, V, 4 * (8 / V) + SHIFT, true, SHIFT>(a, 1024, sms, stream);
}

template <class T>
int run(cudaStream_t stream, const openfish_b200_norm_t *p, int sms) {
    NormArgs<T> a;
    a.x = static_cast<const T *>(p->x); a.r = static_cast<const T *>(p->residual);
    a.w = static_cast<const T *>(p->weight); a.b = static_cast<const T *>(p->bias);
    a.out = static_cast<T *>(p->out); a.q = p->q; a.q_scale = p->q_scale;
    a.x_stride = p->x_stride; a.r_stride = p->residual_stride; a.out_stride = p->out_stride; a.q_stride = p->q_stride;
    a.w_packs = ((uintptr_t)p->weight | (uintptr_t)p->bias) % 16 == 0;
    a.q_packs = (uintptr_t)p->q % 8 == 0 && (p->rows == 1 || p->q_stride % 8 == 0);
    a.rows = p->rows; a.width = p->width; a.kind = p->kind; a.eps = p->eps; a.alpha = p->residual_scale;
    const auto fits = [&](const void *q, long long stride, int to) {
        return !q || ((uintptr_t)q % to == 0 && (p->rows == 1 || stride % 8 == 0));
    };
    // a tensor whose rows all start where x's do between two 16-byte boundaries
    const auto beside = [&](const void *q, long long stride) {
        return !q || (((uintptr_t)q ^ (uintptr_t)p->x) % 16 == 0 && (p->rows == 1 || (stride - p->x_stride) % 8 == 0));
    };
    if (p->width % 8 == 0 && fits(p->x, p->x_stride, 16) && fits(p->residual, p->residual_stride, 16) && fits(p->weight, 0, 16) &&
        fits(p->bias, 0, 16) && fits(p->out, p->out_stride, 16) && fits(p->q, p->q_stride, 8))
        dispatch<T, 8, false>(a, sms, stream);
    else if (beside(p->residual, p->residual_stride) && beside(p->out, p->out_stride))
        dispatch<T, 8, true>(a, sms, stream);
    else
        dispatch<T, 1, false>(a, sms, stream);
    return ofe::launched();
}

}  // namespace

extern "C" int ofb_norm(void *stream, const openfish_b200_norm_t *a) {
    int sms = 0;
    if (const int rc = ofe::sm_count(&sms)) return rc;
    return a->dtype == OPENFISH_B200_F16 ? run<__half>((cudaStream_t)stream, a, sms) : run<__nv_bfloat16>((cudaStream_t)stream, a, sms);
}
