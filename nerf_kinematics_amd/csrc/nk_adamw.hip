// AdamW over many tensors in one launch, with 32-bit or 8-bit moments.
//
//   m <- m + (1 - b1)(g - m)          v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// An 8-bit moment is kept in blocks of 256 consecutive elements of its tensor: one code per element
// (m: OCP e4m3, v: OCP e5m2) and one power-of-two fp32 scale per block, chosen so that the block's
// largest magnitude lies in (2^7, 2^8] (m) or (2^14, 2^15] (v) -- below the format's maximum, so that no
// rounding can overflow.  Codes are rounded stochastically (the part cut off is the probability of
// rounding up): v changes by at most 0.1 % of itself per step at b2 = 0.999, far less than half the
// distance of two codes, and rounding to nearest would never let it decay.  The update itself uses the
// moments before they are rounded.  A positive v never becomes the code 0: m / (sqrt(0) + eps) would
// be a step of m / eps at the next call.
#include <math.h>
#include "nk_common.h"

namespace {

enum { AW_MAX_TENSORS = 56, AW_THREADS = 256, AW_BLOCK = 256, AW_CHUNK = 4 * AW_THREADS,
       AW_MOST = (1 << 24) - 1 };       // workgroups of a launch: fewer than 2^32 threads

// The tensors travel as kernel arguments (no device table to allocate, upload or keep in step with the
// caller's buffers): 56 x 64 bytes + 56 x 4 + scalars stays below the 4 096 bytes of an argument block.
struct AwArgs {
    nk_adamw_tensor t[AW_MAX_TENSORS];
    uint32_t first[AW_MAX_TENSORS];     // first workgroup of each tensor; behind the last tensor: 0xFFFFFFFF
    float omb1, b2, omb2, eps, step_size, bc2_sqrt, decay, gscale;
    uint32_t seed;
    const nk_step_state* st;
};
static_assert(sizeof(AwArgs) <= 4096, "kernel argument block");

template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef float4 type; };
template <> struct Vec4<__bf16> { typedef bf16x4 type; };
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
template <> struct Vec4<_Float16> { typedef f16x4 type; };

template <typename T> NK_D void load4(const T* p, float* o) {
    const auto v = *(const typename Vec4<T>::type*)p;
    o[0] = (float)v.x; o[1] = (float)v.y; o[2] = (float)v.z; o[3] = (float)v.w;
}
template <typename T> NK_D void store4(T* p, const float* o) {
    typename Vec4<T>::type v;
    v.x = (T)o[0]; v.y = (T)o[1]; v.z = (T)o[2]; v.w = (T)o[3];
    *(typename Vec4<T>::type*)p = v;
}
// up to four elements, `live` of them inside the tensor
template <typename T> NK_D void load(const T* p, float* o, bool whole, int live) {
    if (whole) { load4(p, o); return; }
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = k < live ? (float)p[k] : 0.0f;
}
template <typename T> NK_D void store(T* p, const float* o, bool whole, int live) {
    if (whole) { store4(p, o); return; }
#pragma unroll
    for (int k = 0; k < 4; ++k) if (k < live) p[k] = (T)o[k];
}

// Square root to one unit in the last place (v_sqrt_f32), values whose low bits it would drop scaled up first.  The
// step with 8-bit moments is bound by the vector unit, not by memory: this and the factor 1 / sqrt(1 - b2^t)
// in place of a division take about a fifth of its instructions away.
NK_D float root(float v) {
    const bool tiny = v < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(tiny ? v * 0x1p64f : v);
    return tiny ? r * 0x1p-32f : r;
}

// log2 of the scale of a block whose largest magnitude has the bit pattern `bits`: ceil(log2(largest)) - top
NK_D int scale_exp(uint32_t bits, int top) {
    const int e = (int)(bits >> 23) - 127 + ((bits & 0x7FFFFFu) != 0 ? 1 : 0) - top;
    return max(e, -100);
}

// y >= 0 (scaled) to an 8-bit float with MANT fraction bits and exponent bias BIAS, rounded up when the
// part cut off exceeds 1 - r16 / 65536.  Below the smallest normal value the codes are evenly spaced.
template <int MANT, int BIAS> NK_D uint32_t encode(float y, uint32_t r16) {
    constexpr int CUT = 23 - MANT;
    const uint32_t normal = ((__float_as_uint(y) + (r16 << (CUT - 16))) >> CUT) - ((127u - BIAS) << MANT);
    constexpr float SPACING = (float)(1 << (BIAS - 1 + MANT));
    const uint32_t tiny = (uint32_t)__fadd_rn(__fmul_rn(y, SPACING), (float)r16 * (1.0f / 65536.0f));
    return y < 1.0f / (float)(1 << (BIAS - 1)) ? tiny : normal;
}

// One workgroup: AW_CHUNK consecutive elements of one tensor, four consecutive ones a thread, so that a
// wavefront holds exactly one block of 256.  Memory bounds the 32-bit step, memory and the vector unit about
// equally the 8-bit one.  Four elements a thread and many workgroups, not a loop over more: 200 M fp32
// parameters take 1 009 us (5.5 TB/s; a copy reaches 4.8) against 1 067 us with 16 elements a thread, 200 M bf16 ones
// with masters and 8-bit moments 589 us (5.5 TB/s; to 614 us on a warmer card) against 641, the 1.2 M of an 8x256 pair in 48 tensors 7.8 us
// against 11.5.
template <typename PT, typename GT, bool EIGHT>
__global__ __launch_bounds__(AW_THREADS) void k_adamw(const AwArgs A) {
    const int lane = threadIdx.x & 63;
    // the last tensor whose first workgroup is not behind this one
    const uint32_t fb = lane < AW_MAX_TENSORS ? A.first[lane] : 0xFFFFFFFFu;
    const int ti = __popcll(__ballot(fb <= blockIdx.x)) - 1;
    const nk_adamw_tensor& t = A.t[ti];
    const int64_t n = t.n;
    PT* __restrict__ P = (PT*)t.param;
    const GT* __restrict__ G = (const GT*)t.grad;
    float* __restrict__ M32 = (float*)t.exp_avg; float* __restrict__ V32 = (float*)t.exp_avg_sq;
    uint32_t* __restrict__ M8 = (uint32_t*)t.exp_avg; uint32_t* __restrict__ V8 = (uint32_t*)t.exp_avg_sq;
    float* __restrict__ W = t.master;
    float step_size = A.step_size, bc2_sqrt = A.bc2_sqrt, decay = A.decay;
    uint32_t seed = A.seed;
    if (A.st) {
        step_size = A.st->adam_step_size; bc2_sqrt = A.st->adam_bc2_sqrt; decay = 1.0f - A.st->adamw_decay;
        seed = A.st->render_seed;
    }
    const float inv_root = 1.0f / bc2_sqrt;
    const uintptr_t mis = ((uintptr_t)P & (4 * sizeof(PT) - 1)) | ((uintptr_t)G & (4 * sizeof(GT) - 1)) |
                          (((uintptr_t)M32 | (uintptr_t)V32) & (EIGHT ? 3 : 15)) | ((uintptr_t)W & 15);
    const int64_t base = (int64_t)(blockIdx.x - A.first[ti]) * AW_CHUNK;
    const bool whole = mis == 0 && base + AW_CHUNK <= n;
    const int64_t i = base + threadIdx.x * 4;
    const int live = (int)max((int64_t)0, min((int64_t)4, n - i));
    if (base + (threadIdx.x & ~63) * 4 >= n) return;        // wave-uniform: the whole block behind the tensor
    float p[4], g[4], m[4], v[4];
    load(G + i, g, whole, live);
    if (W) load(W + i, p, whole, live); else load(P + i, p, whole, live);
    float sm = 0.0f, sv = 0.0f;
    if (!EIGHT) {
        load(M32 + i, m, whole, live);
        load(V32 + i, v, whole, live);
    } else {
        uint32_t cm = 0, cv = 0;
        if (whole) { cm = M8[i >> 2]; cv = V8[i >> 2]; }
        else for (int k = 0; k < live; ++k) {
            cm |= (uint32_t)((const uint8_t*)M8)[i + k] << (8 * k);
            cv |= (uint32_t)((const uint8_t*)V8)[i + k] << (8 * k);
        }
        sm = t.scale_m[i / AW_BLOCK]; sv = t.scale_v[i / AW_BLOCK];      // i / 256 is in range: the block has a live element
        m[0] = __builtin_amdgcn_cvt_f32_fp8(cm, 0) * sm; m[1] = __builtin_amdgcn_cvt_f32_fp8(cm, 1) * sm;
        m[2] = __builtin_amdgcn_cvt_f32_fp8(cm, 2) * sm; m[3] = __builtin_amdgcn_cvt_f32_fp8(cm, 3) * sm;
        v[0] = __builtin_amdgcn_cvt_f32_bf8(cv, 0) * sv; v[1] = __builtin_amdgcn_cvt_f32_bf8(cv, 1) * sv;
        v[2] = __builtin_amdgcn_cvt_f32_bf8(cv, 2) * sv; v[3] = __builtin_amdgcn_cvt_f32_bf8(cv, 3) * sv;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float gk = g[k] * A.gscale;
        m[k] = __fadd_rn(m[k], __fmul_rn(gk - m[k], A.omb1));
        v[k] = __fadd_rn(__fmul_rn(v[k], A.b2), __fmul_rn(A.omb2, __fmul_rn(gk, gk)));
        const float denom = root(v[k]) * inv_root + A.eps;
        p[k] = __fsub_rn(__fmul_rn(p[k], decay), __fmul_rn(m[k] / denom, step_size));
    }
    if (W) store(W + i, p, whole, live);
    store(P + i, p, whole, live);
    if (!EIGHT) {
        store(M32 + i, m, whole, live);
        store(V32 + i, v, whole, live);
    } else {
        uint32_t bm = 0, bv = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) if (k < live) {
            bm = max(bm, __float_as_uint(m[k]) & 0x7FFFFFFFu);
            bv = max(bv, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        }
        bm = nk_wave_max(bm); bv = nk_wave_max(bv);
        const int em = scale_exp(bm, 8), ev = scale_exp(bv, 15);
        const float im = __uint_as_float((uint32_t)(127 - em) << 23), iv = __uint_as_float((uint32_t)(127 - ev) << 23);
        uint32_t cm = 0, cv = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t r = nk_rand_u32(seed, NK_STREAM_OPTIMISER, (uint64_t)(i + k));
            const uint32_t qm = encode<3, 7>(fabsf(m[k]) * im, r & 0xFFFFu) | (m[k] < 0.0f ? 0x80u : 0u);
            uint32_t qv = encode<2, 15>(v[k] * iv, r >> 16);
            if (qv == 0 && v[k] > 0.0f) qv = 1;
            cm |= (qm & 0xFFu) << (8 * k); cv |= (qv & 0xFFu) << (8 * k);
        }
        if (whole) { M8[i >> 2] = cm; V8[i >> 2] = cv; }
        else for (int k = 0; k < live; ++k) {
            ((uint8_t*)M8)[i + k] = (uint8_t)(cm >> (8 * k));
            ((uint8_t*)V8)[i + k] = (uint8_t)(cv >> (8 * k));
        }
        if (lane == 0) {        // a block that holds an infinity or a NaN decodes to NaN
            t.scale_m[i / AW_BLOCK] = bm >= 0x7F800000u ? __builtin_nanf("") : __uint_as_float((uint32_t)(127 + em) << 23);
            t.scale_v[i / AW_BLOCK] = bv >= 0x7F800000u ? __builtin_nanf("") : __uint_as_float((uint32_t)(127 + ev) << 23);
        }
    }
}

template <typename PT, typename GT> void launch(bool eight, unsigned blocks, hipStream_t st, const AwArgs& a) {
    if (eight) hipLaunchKernelGGL((k_adamw<PT, GT, true>), dim3(blocks), dim3(AW_THREADS), 0, st, a);
    else hipLaunchKernelGGL((k_adamw<PT, GT, false>), dim3(blocks), dim3(AW_THREADS), 0, st, a);
}

}  // namespace

extern "C" int nk_adamw_step(const nk_adamw_tensor* tensors, int32_t count, const nk_adamw_opts* o, void* stream) {
    if (!o || count < 0 || (count > 0 && !tensors)) NK_FAIL(NK_ERR_ARG, "nk_adamw_step: null pointer or count < 0");
    const int pd = o->param_dtype, gd = o->grad_dtype;
    if (pd < NK_F32 || pd > NK_F16 || gd < NK_F32 || gd > NK_F16) NK_FAIL(NK_ERR_ARG, "nk_adamw_step: unknown dtype %d / %d", pd, gd);
    if (gd != pd && gd != NK_F32) NK_FAIL(NK_ERR_UNSUPPORTED, "nk_adamw_step: gradients of dtype %d with parameters of dtype %d (fp32 or the same)", gd, pd);
    if (o->state_bits != 32 && o->state_bits != 8) NK_FAIL(NK_ERR_UNSUPPORTED, "nk_adamw_step: state_bits=%d (32 | 8)", o->state_bits);
    if (!o->state && o->step < 1) NK_FAIL(NK_ERR_ARG, "nk_adamw_step: step < 1");
    if (!(o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0 && o->eps >= 0.0))
        NK_FAIL(NK_ERR_ARG, "nk_adamw_step: beta1, beta2 in [0, 1) and eps >= 0 wanted");
    const bool eight = o->state_bits == 8;
    for (int32_t k = 0; k < count; ++k) {
        const nk_adamw_tensor& t = tensors[k];
        if (t.n < 0) NK_FAIL(NK_ERR_ARG, "nk_adamw_step: tensor %d has a negative size", k);
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (eight && (!t.scale_m || !t.scale_v)))
            NK_FAIL(NK_ERR_ARG, "nk_adamw_step: null pointer in tensor %d", k);
        if (t.n > (int64_t)AW_CHUNK * AW_MOST) NK_FAIL(NK_ERR_UNSUPPORTED, "nk_adamw_step: tensor %d is too large", k);
    }
    AwArgs a;
    a.omb1 = (float)(1.0 - o->beta1); a.b2 = (float)o->beta2; a.omb2 = (float)(1.0 - o->beta2); a.eps = (float)o->eps;
    a.step_size = a.decay = 0.0f; a.bc2_sqrt = 1.0f;
    if (!o->state) {
        a.step_size = (float)(o->lr / (1.0 - pow(o->beta1, (double)o->step)));
        a.bc2_sqrt = (float)sqrt(1.0 - pow(o->beta2, (double)o->step));
        a.decay = 1.0f - (float)(o->lr * o->weight_decay);         // as the kernel forms it from *state
    }
    a.gscale = o->grad_scale; a.seed = o->seed; a.st = o->state;
    int32_t k = 0;
    while (k < count) {
        int held = 0;
        uint64_t blocks = 0;
        for (; k < count && held < AW_MAX_TENSORS; ++k) {
            if (tensors[k].n == 0) continue;
            const uint64_t more = (uint64_t)((tensors[k].n + AW_CHUNK - 1) / AW_CHUNK);
            if (held > 0 && blocks + more > AW_MOST) break;
            a.t[held] = tensors[k]; a.first[held] = (uint32_t)blocks;
            blocks += more; ++held;
        }
        if (held == 0) break;
        for (int j = held; j < AW_MAX_TENSORS; ++j) { a.t[j] = nk_adamw_tensor{}; a.first[j] = 0xFFFFFFFFu; }
        const hipStream_t st = nk_stream(stream);
        if (pd == NK_F32) launch<float, float>(eight, (unsigned)blocks, st, a);
        else if (pd == NK_BF16) { if (gd == NK_F32) launch<__bf16, float>(eight, (unsigned)blocks, st, a); else launch<__bf16, __bf16>(eight, (unsigned)blocks, st, a); }
        else { if (gd == NK_F32) launch<_Float16, float>(eight, (unsigned)blocks, st, a); else launch<_Float16, _Float16>(eight, (unsigned)blocks, st, a); }
        NK_CHECK_LAUNCH("k_adamw");
    }
    return NK_OK;
}
