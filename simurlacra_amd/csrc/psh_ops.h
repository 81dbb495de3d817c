// What the translation units of the policy operators (ops_linear.hip, ops_memory.hip) share: element types, the search
// for the part of the rows that a workgroup works on (its arithmetic: psh_parts.h), and the fp32 / fp64 elementary functions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "psh_ctx.h"
#include "psh_math.h"
#include "psh_parts.h"

#define PSH_OP __device__ __forceinline__

typedef unsigned short bf16_t;  // storage; arithmetic is fp32
typedef float v4f __attribute__((ext_vector_type(4)));
typedef double v4d __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

template <class T> struct Wide { typedef float type; };
template <> struct Wide<double> { typedef double type; };

PSH_OP float to_wide(bf16_t x) { return __uint_as_float((unsigned)x << 16); }
PSH_OP float to_wide(float x) { return x; }
PSH_OP double to_wide(double x) { return x; }
// to the nearest, ties to even; a NaN stays one.  The hardware conversion (v_cvt_pk_bf16_f32) rounds the same way.
template <class T> PSH_OP T to_elem(typename Wide<T>::type x);
template <> PSH_OP float to_elem<float>(float x) { return x; }
template <> PSH_OP double to_elem<double>(double x) { return x; }
template <> PSH_OP bf16_t to_elem<bf16_t>(float x) {
    const __bf16 b = (__bf16)x;
    return __builtin_bit_cast(bf16_t, b);
}

// ------------------------------------------------------------------------------------------ elementary functions
// Without branches, so that the elements a lane works on run side by side; NaN arguments give NaNs by themselves.
// fp32: v_exp_f32 / v_log_f32 / v_rcp_f32 are within 1 ulp of the power, logarithm and reciprocal; what the argument's
// scaling by log2(e) adds is |x| 2^-24 relative, which an exponential of a negative argument shrinks again.
// fp64: psh_exp's core, which is right, and over- or underflows, for every |x| < 2^30; only the high word of what lies
// beyond is replaced (a NaN compares false and stays one).
#define PSH_LOG2E 1.4426950408889634
#define PSH_LN2 0.6931471805599453
PSH_OP float exp2_w(float x) { return __builtin_amdgcn_exp2f(x); }
PSH_OP float exp_w(float x) { return __builtin_amdgcn_exp2f(x * (float)PSH_LOG2E); }
PSH_OP double exp_w(double x) {
    const int hi = __double2hiint(x);
    return psh_exp_core(__hiloint2double(fabs(x) > 1e9 ? (hi & (int)0x80000000) | 0x41cdcd65 : hi, __double2loint(x)));
}
PSH_OP float rcp_w(float x) { return __builtin_amdgcn_rcpf(x); }
PSH_OP float sigmoid_w(float x) { return rcp_w(1.f + exp_w(-x)); }
PSH_OP double sigmoid_w(double x) {
    const double e = exp_w(-fabs(x)), r = psh_rcp_refined(1. + e);   // (the denominator lies in [1, 2])
    return x >= 0. ? r : e * r;
}
template <class W> PSH_OP W silu_w(W x) { return x * sigmoid_w(x); }
// d/dx of x sigmoid(x) from s = sigmoid(x)
template <class W> PSH_OP W silu_slope_w(W x, W s) { return s * (W(1) + x * (W(1) - s)); }
// log(1 + e^x) = max(x, 0) + log1p(e^-|x|).  log1p keeps the digits of a small e, where the step sizes of a slow memory are:
// w = 1 + e rounds, and e - (w - 1) is what that lost, exactly; it goes back in front of log's slope 1 / w, which is 1 where
// it matters (for e near 1 the lost part is below half a ulp of the result anyway).
PSH_OP float softplus_w(float x) {
    const float e = exp_w(-fabsf(x)), w = 1.f + e;
    return fmaxf(x, 0.f) + (__builtin_amdgcn_logf(w) * (float)PSH_LN2 + (e - (w - 1.f)));
}
PSH_OP double softplus_w(double x) {
    const double e = exp_w(-fabs(x)), w = 1. + e;
    return fmax(x, 0.) + (psh_log_normal(w) + (e - (w - 1.)));
}
// the same and its derivative, sigmoid(x), from one exponential
PSH_OP float softplus_w(float x, float& slope) {
    const float e = exp_w(-fabsf(x)), w = 1.f + e, r = rcp_w(w);
    slope = x >= 0.f ? r : e * r;
    return fmaxf(x, 0.f) + (__builtin_amdgcn_logf(w) * (float)PSH_LN2 + (e - (w - 1.f)));
}
PSH_OP double softplus_w(double x, double& slope) {
    const double e = exp_w(-fabs(x)), w = 1. + e, r = psh_rcp_refined(w);
    slope = x >= 0. ? r : e * r;
    return fmax(x, 0.) + (psh_log_normal(w) + (e - (w - 1.)));
}
// x where the mask is all ones, 0 where it is 0, whatever x is
PSH_OP float masked(float x, int mask) { return __int_as_float(__float_as_int(x) & mask); }
PSH_OP double masked(double x, int mask) { return __hiloint2double(__double2hiint(x) & mask, __double2loint(x) & mask); }
PSH_OP float tanh_w(float x) { return tanhf(x); }
PSH_OP double tanh_w(double x) { return psh_tanh(x); }

// derivative of the nonlinearity from its value
template <class W> PSH_OP W nonlin_slope_w(int kind, W y) {
    if (kind == PSH_NL_TANH) return W(1) - y * y;
    if (kind == PSH_NL_SIGMOID) return y * (W(1) - y);
    if (kind == PSH_NL_RELU) return y <= W(0) ? W(0) : W(1);
    return W(1);
}

// ------------------------------------------------------------------------------------------ parts of the rows
template <class F> PSH_OP int wave_search(int n, int slot, F key) {
    const int lane = __lane_id();
    Search s{0, n + 1};
    while (s.count > 1) {
        const int i = s.candidate(lane);
        s.narrow(__ballot(s.probes(lane) && key(i) <= slot));
    }
    return __builtin_amdgcn_readfirstlane(s.lo);
}

PSH_OP Piece find_piece(const Parts& p, int slot) {
    const int part = wave_search(p.n, slot, [&](int i) { return p.first_slot(i); });
    return piece_of(p, part, __builtin_amdgcn_readfirstlane(p.at(part)), __builtin_amdgcn_readfirstlane(p.at(part + 1)), slot);
}

// ------------------------------------------------------------------------------------------ host side
// the calling thread's current device is the context's for the duration of a call
struct DeviceScope {
    int before = -1;
    bool ok = false;
    explicit DeviceScope(int device) {
        ok = hipGetDevice(&before) == hipSuccess && (before == device || hipSetDevice(device) == hipSuccess);
        if (before == device) before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
#define PSH_ON_DEVICE(ctx)                                                         \
    DeviceScope scope_((ctx)->device);                                             \
    if (!scope_.ok) {                                                              \
        set_err(ctx, "cannot make the context's GPU current");                     \
        return PSH_ERR_HIP;                                                        \
    }
