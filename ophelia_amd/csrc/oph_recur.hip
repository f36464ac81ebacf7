// Gated linear recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t, a = sigmoid(gate), and its gradient: oph_seq_recur_forward / _gradient.
//
// Every step is an affine map of the state, and maps compose: (A, B) then (A', B') is (A'A, A'B + B').  A workgroup owns 128 bytes of
// channels of one sequence and goes over time in blocks of 32 stretches of R steps: each thread runs its stretch from 0, the maps are
// composed over the 8 stretches of a wave by lane exchanges and over the 4 waves through LDS, and the thread runs its stretch once
// more from the state it now knows.  The inputs stay in registers in between: one pass over memory.
// Gradient, backwards in time with the map m_t = a_t (m_{t+1} + dh_t):  l_t = dh_t + m_{t+1}, dx = (1 - a) l, dgate = a (1 - a) (h_{t-1} - x) l.
#include "oph_seq.h"
#include "../../include/ophelia_hip.h"

#include <algorithm>

namespace ophseq {

struct RecurP {
    const void *x, *gate, *hin, *dh;
    const float *h0, *dh_last;
    void *h, *dx, *dgate;
    float *h_last, *dh0;
    const int* lens;
    int64_t xs[2], gs[2], hs[2], ds[2];
    int B, T, C;
};

template <class T> struct Piece {                                     // 16 bytes of channels, `left` of the row's remain
    static constexpr int PER = El<T>::PER16;
    typedef T vec __attribute__((ext_vector_type(PER)));
    static __device__ __forceinline__ u32x4 load(const T* at, int left) {
        if (left >= PER) return load16(at);
        vec v;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = j < left ? at[j] : (T)0.f;
        return __builtin_bit_cast(u32x4, v);
    }
    static __device__ __forceinline__ void store(T* at, const float (&f)[PER], int left) {
        vec v;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = (T)f[j];
        if (left >= PER) store16(at, __builtin_bit_cast(u32x4, v));
        else
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (j < left) at[j] = v[j];
    }
    static __device__ __forceinline__ float at(u32x4 x, int j) { return (float)__builtin_bit_cast(vec, x)[j]; }
};

// sigmoid and 1 - sigmoid, each without cancellation: a state that is held for thousands of steps has 1 - a of 1e-4 and less
__device__ __forceinline__ void gate_of(float g, float& a, float& keep) {
    const float e = exp2_(-fabsf(g) * LOG2E), r = __builtin_amdgcn_rcpf(1.f + e);
    a = g >= 0.f ? r : e * r;
    keep = g >= 0.f ? e * r : r;
}

// Maps (A, B) of this thread's stretch and the state before the block -> the state before the stretch; `state` moves behind the block
template <int PER>
__device__ __forceinline__ void compose(float (&A)[PER], float (&B)[PER], float (&state)[PER], float (&in)[PER], float (*lds)[8][PER][2], int lane, int wave) {
#pragma unroll
    for (int off = 8; off < 64; off <<= 1)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float a = __shfl_up(A[j], off), b = __shfl_up(B[j], off);
            if (lane >= off) {
                B[j] = fmaf(A[j], b, B[j]);
                A[j] *= a;
            }
        }
    if (lane >= 56)
#pragma unroll
        for (int j = 0; j < PER; ++j) { lds[wave][lane & 7][j][0] = A[j]; lds[wave][lane & 7][j][1] = B[j]; }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        float a = __shfl_up(A[j], 8), b = __shfl_up(B[j], 8);
        if (lane < 8) { a = 1.f; b = 0.f; }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w == wave) in[j] = fmaf(a, state[j], b);
            state[j] = fmaf(lds[w][lane & 7][j][0], state[j], lds[w][lane & 7][j][1]);
        }
    }
}

template <class T> __global__ __launch_bounds__(256) void recur_forward(const RecurP p) {
    constexpr int PER = El<T>::PER16, R = 8, BLOCK = 32 * R;
    __shared__ float lds[2][4][8][PER][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = threadIdx.x >> 3;
    const int slabs = (p.C + 8 * PER - 1) / (8 * PER), b = blockIdx.x / slabs;
    const int c = ((blockIdx.x - b * slabs) * 8 + (lane & 7)) * PER, left = p.C - c;
    const int len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
    const int cc = left > 0 ? c : 0, cl = left > 0 ? left : p.C;        // lanes beyond the channels read the first ones and write nothing
    const T* x = (const T*)p.x + b * p.xs[0] + cc;
    const T* g = (const T*)p.gate + b * p.gs[0] + cc;
    T* h = (T*)p.h + (int64_t)b * p.T * p.C + cc;
    float state[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) state[j] = p.h0 && j < left ? p.h0[(int64_t)b * p.C + c + j] : 0.f;
    int k = 0, t0 = 0;
    for (; t0 < len; t0 += BLOCK, ++k) {
        const int t = t0 + sub * R;
        u32x4 xr[R], gr[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t tt = min(t + r, len - 1);
            xr[r] = Piece<T>::load(x + tt * p.xs[1], cl);
            gr[r] = Piece<T>::load(g + tt * p.gs[1], cl);
        }
        float A[PER], B[PER], s[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            A[j] = 1.f;
            B[j] = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float a, keep;
                gate_of(Piece<T>::at(gr[r], j), a, keep);
                if (t + r < len) {
                    A[j] *= a;
                    B[j] = fmaf(a, B[j], keep * Piece<T>::at(xr[r], j));
                }
            }
        }
        compose<PER>(A, B, state, s, lds[k & 1], lane, wave);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float out[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                float a, keep;
                gate_of(Piece<T>::at(gr[r], j), a, keep);
                s[j] = fmaf(a, s[j], keep * Piece<T>::at(xr[r], j));
                out[j] = t + r < len ? s[j] : 0.f;
            }
            if (t + r < p.T && left > 0) Piece<T>::store(h + (int64_t)(t + r) * p.C, out, left);
        }
    }
    const float zero[PER] = {};
    for (int t = t0 + sub; t < p.T; t += 32)
        if (left > 0) Piece<T>::store(h + (int64_t)t * p.C, zero, left);
    if (sub == 0)
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j < left) p.h_last[(int64_t)b * p.C + c + j] = state[j];
}

template <class T> __global__ __launch_bounds__(256) void recur_gradient(const RecurP p) {
    constexpr int PER = El<T>::PER16, R = 8, BLOCK = 32 * R;
    __shared__ float lds[2][4][8][PER][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = threadIdx.x >> 3;
    const int slabs = (p.C + 8 * PER - 1) / (8 * PER), b = blockIdx.x / slabs;
    const int c = ((blockIdx.x - b * slabs) * 8 + (lane & 7)) * PER, left = p.C - c;
    const int len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
    const int cc = left > 0 ? c : 0, cl = left > 0 ? left : p.C;
    const T* x = (const T*)p.x + b * p.xs[0] + cc;
    const T* g = (const T*)p.gate + b * p.gs[0] + cc;
    const T* h = (const T*)p.hin + b * p.hs[0] + cc;
    const T* d = (const T*)p.dh + b * p.ds[0] + cc;
    T* dx = (T*)p.dx + (int64_t)b * p.T * p.C + cc;
    T* dg = (T*)p.dgate + (int64_t)b * p.T * p.C + cc;
    float state[PER], first[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        state[j] = p.dh_last && j < left ? p.dh_last[(int64_t)b * p.C + c + j] : 0.f;
        first[j] = p.h0 && j < left ? p.h0[(int64_t)b * p.C + c + j] : 0.f;
    }
    int k = 0;
    for (int u0 = 0; u0 < len; u0 += BLOCK, ++k) {
        const int t = len - 1 - u0 - sub * R;                            // this thread: t, t-1, ..., t-R+1
        u32x4 xr[R], gr[R], hr[R], dr[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t tt = max(t - r, 0);
            xr[r] = Piece<T>::load(x + tt * p.xs[1], cl);
            gr[r] = Piece<T>::load(g + tt * p.gs[1], cl);
            dr[r] = Piece<T>::load(d + tt * p.ds[1], cl);
            hr[r] = Piece<T>::load(h + max(tt - 1, (int64_t)0) * p.hs[1], cl);
        }
        float A[PER], B[PER], s[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            A[j] = 1.f;
            B[j] = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float a, keep;
                gate_of(Piece<T>::at(gr[r], j), a, keep);
                if (t - r >= 0) {
                    A[j] *= a;
                    B[j] = a * (B[j] + Piece<T>::at(dr[r], j));
                }
            }
        }
        compose<PER>(A, B, state, s, lds[k & 1], lane, wave);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float ox[PER], og[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                float a, keep;
                gate_of(Piece<T>::at(gr[r], j), a, keep);
                const float l = Piece<T>::at(dr[r], j) + s[j];
                const float before = t - r > 0 ? Piece<T>::at(hr[r], j) : first[j];
                ox[j] = keep * l;
                og[j] = a * keep * (before - Piece<T>::at(xr[r], j)) * l;
                s[j] = a * l;
            }
            if (t - r >= 0 && left > 0) {
                Piece<T>::store(dx + (int64_t)(t - r) * p.C, ox, left);
                Piece<T>::store(dg + (int64_t)(t - r) * p.C, og, left);
            }
        }
    }
    const float zero[PER] = {};
    for (int t = len + sub; t < p.T; t += 32)
        if (left > 0) {
            Piece<T>::store(dx + (int64_t)t * p.C, zero, left);
            Piece<T>::store(dg + (int64_t)t * p.C, zero, left);
        }
    if (sub == 0 && p.dh0)
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j < left) p.dh0[(int64_t)b * p.C + c + j] = state[j];
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------------
static int check(const oph_seq_recur* a) {
    if (!a) return fail(OPH_ERR_INVALID, "recurrence: no arguments");
    if (!type_bytes(a->dtype)) return fail(OPH_ERR_INVALID, "recurrence: dtype %d is not one of OPH_SEQ_*", a->dtype);
    if (a->B < 0 || a->T < 0 || a->C < 1) return fail(OPH_ERR_INVALID, "recurrence: bad size (B %d, T %d, C %d)", a->B, a->T, a->C);
    if (a->T > 2147483647 - 4096 || a->C > 1 << 28 || (double)a->B * (a->C / 32 + 1) > 2.0e9)
        return fail(OPH_ERR_UNSUPPORTED, "recurrence: too large (B %d, T %d, C %d)", a->B, a->T, a->C);
    return OPH_OK;
}
static RecurP params(const oph_seq_recur* a) {
    RecurP p = {};
    p.x = a->x; p.gate = a->gate; p.h0 = a->h0; p.lens = a->lens;
    p.B = a->B; p.T = a->T; p.C = a->C;
    for (int i = 0; i < 2; ++i) { p.xs[i] = a->x_stride[i]; p.gs[i] = a->gate_stride[i]; p.hs[i] = a->h_stride[i]; p.ds[i] = a->dh_stride[i]; }
    return p;
}
template <class T> static dim3 grid(const RecurP& p) { return dim3((unsigned)(p.B * cdiv(p.C, 8 * El<T>::PER16))); }

}  // namespace ophseq

using namespace ophseq;
extern "C" {

int64_t oph_seq_recur_workspace(const oph_seq_recur* a, int gradient) {
    (void)gradient;
    if (int rc = check(a)) return rc;
    return 0;
}

int oph_seq_recur_forward(const oph_seq_recur* a, int device, void* stream) {
    if (int rc = check(a)) return rc;
    if (!a->B) return OPH_OK;
    if (!a->h_last || (a->T && (!a->x || !a->gate || !a->h))) return fail(OPH_ERR_INVALID, "recurrence: x, gate, h and h_last must not be NULL");
    OnDevice on(device);
    if (on.status) return on.status;
    RecurP p = params(a);
    p.h = a->h;
    p.h_last = a->h_last;
    if (a->dtype == OPH_SEQ_F32) return launch<RecurP>(recur_forward<float>, grid<float>(p), 256, p, 0, stream);
    if (a->dtype == OPH_SEQ_BF16) return launch<RecurP>(recur_forward<bf16_t>, grid<bf16_t>(p), 256, p, 0, stream);
    return launch<RecurP>(recur_forward<f16_t>, grid<f16_t>(p), 256, p, 0, stream);
}

int oph_seq_recur_gradient(const oph_seq_recur* a, int device, void* stream) {
    if (int rc = check(a)) return rc;
    if (!a->B) return OPH_OK;
    if (a->T && (!a->x || !a->gate || !a->h || !a->dh || !a->dx || !a->dgate))
        return fail(OPH_ERR_INVALID, "recurrence: x, gate, h, dh, dx and dgate must not be NULL");
    OnDevice on(device);
    if (on.status) return on.status;
    RecurP p = params(a);
    p.hin = a->h; p.dh = a->dh; p.dh_last = a->dh_last; p.dx = a->dx; p.dgate = a->dgate; p.dh0 = a->dh0;
    if (a->dtype == OPH_SEQ_F32) return launch<RecurP>(recur_gradient<float>, grid<float>(p), 256, p, 0, stream);
    if (a->dtype == OPH_SEQ_BF16) return launch<RecurP>(recur_gradient<bf16_t>, grid<bf16_t>(p), 256, p, 0, stream);
    return launch<RecurP>(recur_gradient<f16_t>, grid<f16_t>(p), 256, p, 0, stream);
}

}  // extern "C"
