// Cross attention, gradient: oph_seq_attn_gradient.
//
// Two passes, each of which owns what it writes, so that no sum depends on an order of arrival: attn_dq (a workgroup owns 128 rows and
// runs over the keys) also forms delta = dout.out for attn_dkv (a workgroup owns 128 keys and runs over the rows).  Both recompute the
// scores from q, k and the forward's lse: 7 products of Tq x Tk x D instead of 5, for nothing to add up across workgroups.
#include "oph_attn.h"
#include "../../include/ophelia_hip.h"

#include <math.h>

namespace ophseq {

__device__ __forceinline__ float dot8(f32x8 a, f32x8 b) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(a[j], b[j], s);
    return s;
}

// Score gradients dS = P (dP - delta) are rounded to the operand type of the next product.  float16 ends at 65504, which they can pass where the
// gradients that they are summed to do not: every column of a result has a power of two `by` that its dS are multiplied by and that is taken out
// at the end, both exactly; 1 unless they can pass 2^15.
// dq, whose column is a query: `by` is lowered when a dS asks for it, and what has been summed is brought to the new one (the running maximum of a
// softmax, in steps of 2).
template <class T, int N> __device__ __forceinline__ void into_range(f32x16& S, float& by, f32x16 (&acc)[N]) {
    if constexpr (__is_same(T, f16_t)) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(S[i]));
        if (__any(top * by > 32768.f)) {
            top = fmaxf(top, other_half(top));                              // both halves hold elements of the column
            const float now = top * by > 32768.f && top < INFINITY ? ldexpf(1.f, 14 - ilogbf(top)) : by;      // what is infinite stays so
            const float f = now / by;
#pragma unroll
            for (int d = 0; d < N; ++d) acc[d] *= f;
            by = now;
        }
        if (__any(by != 1.f)) S *= by;
    }
}
// dk, whose column is a key (its D > 128 form has no register left for that): |dS| <= |dout of the row| |v of the key| + |delta|, since P <= 1.  attn_dq
// leaves the largest |dout| and |delta| of every 32 rows behind delta, and the bound is known before the first product.  It may be
// far above the largest dS; what that costs lies below 2^-25 of the bound's 2^15, a 2^-40th of it.  Together (2 x 16 heads over 4 key heads of
// 4096 x 4096 fp16): x 128 1000 -> 1060 us, x 256 unchanged; dk lowered as dq is spilled 265 registers at x 256, 4010 -> 7600.
template <class T> __device__ __forceinline__ float* range_of(const AttnP& p, const Where& w, int tiles) {
    return p.aux + ((int64_t)p.B * p.Hk * p.G * p.Tq + 3) / 4 * 4 + (int64_t)(w.b * p.Hk + w.hk) * tiles * 8;
}
template <class T, int N> __device__ __forceinline__ float norm_of(const frag_t<T> (&x)[N]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += dot8(__builtin_convertvector(x[i], f32x8), __builtin_convertvector(x[i], f32x8));
    return sqrtf(s + other_half(s));
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x = fmaxf(x, __shfl_xor(x, i));
    return x;
}

// ---- dq: S^T = K q^T and dP^T = V dout^T have the queries as columns; dS^T is the operand of dq^T = K^T dS^T -------------------------------
// 16 bits: waves a SIMD that the registers must leave room for, and rows of a tile in LDS -- D = 64 has few products between two barriers
// (2 x 16 heads of 4096 x 4096 x 64: 499 us, with tiles of 32 rows 608).
template <class T, int DP> constexpr int grad_waves(int of64) { return sizeof(T) == 4 || DP > 128 ? 1 : DP > 64 ? 2 : of64; }
template <class T, int DP> constexpr int grad_tile() { return sizeof(T) == 2 && DP == 64 ? 64 : 32; }
template <class T, int DP>
__global__ __launch_bounds__(256, (grad_waves<T, DP>(3))) void attn_dq(const AttnP p) {
    constexpr int KT = grad_tile<T, DP>(), TB = Tile<T, DP>::bytes(KT);
    constexpr uint64_t FULL = KT == 64 ? ~0ull : 0xffffffffull;
    __shared__ __attribute__((aligned(16))) char lds[4 * TB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
    const int M = p.Tq * p.G, Hq = p.Hk * p.G, tiles = (M + 127) / 128;
    const int lin = on_xcd(p, blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int r = w.tile * 128 + wave * 32 + col, t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
    const bool row = r < M && t < w.qlen;
    const float c = p.scale * LOG2E;

    const T* k = (const T*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const T* v = (const T*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    const Span span = split_span(w.klen, KT, p.nsplit, split, row_time(p, w.tile * 128) < w.qlen);
    const int kbeg = span.beg, kend = span.end;
    const int nt = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;
    Stage<T, DP, KT, 256> sk, sv;
    const T *k1 = sk.own(k + kbeg * p.ks[1], p.ks[1], p.D, tid), *v1 = sv.own(v + kbeg * p.vs[1], p.vs[1], p.D, tid);
    uint64_t bits = 0;
    uint8_t byte = 0;
    auto fetch = [&](int j) {
        const int key0 = kbeg + j * KT, last = kend - 1;
        byte = key_byte(p, w, key0, kend, lane);
        if (key0 + KT <= kend) {
            sk.load_run(k1, p.ks[1]);
            sv.load_run(v1, p.vs[1]);
            k1 += KT * p.ks[1];
            v1 += KT * p.vs[1];
            return;
        }
        sk.load([&](int i) { return k + (int64_t)min(key0 + i, last) * p.ks[1]; }, p.D, tid);
        sv.load([&](int i) { return v + (int64_t)min(key0 + i, last) * p.vs[1]; }, p.D, tid);
    };
    auto commit = [&](int j) {
        char* x = lds + (j & 1) * 2 * TB;
        bits = key_bits(byte, kbeg + j * KT, kend, lane) & FULL;
        sk.store(x, bits, p.D, tid);
        sv.store(x + TB, bits, p.D, tid);
    };
    if (nt) fetch(0);                                    // on its way while the rows' operands are loaded

    frag_t<T> Q[DP / 16], dO[DP / 16];
    f32x16 dQ[DP / 32];
    row_frags<T, DP>(Q, row_ptr<T>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]), p.D, row, half);
    row_frags<T, DP>(dO, row_ptr<T>(p, p.dout, w, r, p.ds[0], p.ds[1], p.ds[2]), p.D, row, half);
    float delta = 0.f, lse2 = INFINITY;                   // exp2(s - inf) = 0: rows that are not there or that saw no key
    {
        const T* o = row_ptr<T>(p, p.out, w, r, (int64_t)p.Tq * Hq * p.D, (int64_t)Hq * p.D, p.D);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int d = s * 16 + half * 8;
            const T* at = o + (d < p.D ? d : 0);
            const frag_t<T> x = bits_to_frag<T>(load16(at), sizeof(T) == 4 ? load16(at + 4) : u32x4{0, 0, 0, 0});
            delta += dot8(__builtin_convertvector(x, f32x8), __builtin_convertvector(dO[s], f32x8));
        }
        delta += other_half(delta);
        if (!row) delta = 0.f;
        const int64_t at = ((int64_t)w.b * Hq + h) * p.Tq + t;
        if (row) {
            const float lse = p.lse[at];
            if (lse != -INFINITY) lse2 = lse * LOG2E;
        }
        if (r < M && half == 0 && split == 0) p.aux[at] = delta;
        if constexpr (__is_same(T, f16_t))
            if (split == 0) {
                const float n = wave_max(norm_of<T>(dO)), d = wave_max(fabsf(delta));
                float* to = range_of<T>(p, w, tiles) + (w.tile * 4 + wave) * 2;
                if (lane == 0) { to[0] = n; to[1] = d; }
            }
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dQ[d] = f32x16{};
    float by = 1.f;

    if (nt) commit(0);
    for (int j = 0; j < nt; ++j) {
        const uint64_t now = bits;
        __syncthreads();
        if (j + 1 < nt) fetch(j + 1);
        if (now) {
            const char *tk = lds + (j & 1) * 2 * TB, *tv = tk + TB;
#pragma unroll
            for (int k0 = 0; k0 < KT; k0 += 32) {
                f32x16 S = {}, dP = {};
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) {
                    S = El<T>::mma(row_frag<T, DP>(tk, k0, s, lane), Q[s], S);
                    dP = El<T>::mma(row_frag<T, DP>(tv, k0, s, lane), dO[s], dP);
                }
                const uint32_t b = (uint32_t)(now >> k0) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) S[i] = exp2_(fmaf(S[i], c, -lse2)) * (dP[i] - delta);
                if (now != FULL) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = (b >> (8 * (i / 4) + i % 4)) & 1 ? S[i] : 0.f;
                }
                into_range<T>(S, by, dQ);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const frag_t<T> dS = next_frag<T>(S, s);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) dQ[d] = El<T>::mma(trans_frag<T, DP>(tk, k0 + 16 * s, 32 * d, lane), dS, dQ[d]);
                }
            }
        }
        if (j + 1 < nt) commit(j + 1);
    }

    if (r < M) {
        const int64_t at = (((int64_t)w.b * p.Tq + t) * Hq + h) * p.D;
        T* o = (T*)p.o0 + at;
        float* part = p.part + (int64_t)split * p.B * p.Tq * Hq * p.D + at;
        const float f = p.scale / by;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int e = 32 * d + 8 * g + 4 * half;
                f32x4 x = {dQ[d][4 * g], dQ[d][4 * g + 1], dQ[d][4 * g + 2], dQ[d][4 * g + 3]};
                x = row ? x * f : f32x4{0.f, 0.f, 0.f, 0.f};
                if (e < p.D) {
                    if (p.nsplit == 1) store4<T>(o + e, x);
                    else *(f32x4*)(part + e) = x;
                }
            }
    }
}

// ---- dk, dv: S = q K^T and dP = dout V^T have the keys as columns; P and dS are the operands of dv^T = dout^T P and dk^T = q^T dS.
// BOTH: one workgroup forms both.  Otherwise (D > 128: both results and both key operands do not fit the registers) half of the grid
// forms dv and half dk, and the scores are formed twice. ----
template <class T, int DP, bool BOTH>
__global__ __launch_bounds__(256, (grad_waves<T, DP>(2))) void attn_dkv(const AttnP p) {
    constexpr int RT = grad_tile<T, DP>(), TB = Tile<T, DP>::bytes(RT), TV = Tile<T, DP>::bytes(32), NACC = BOTH ? 2 : 1;
    // 16 bits, D = 128: with the values' operand in LDS too the rest fits the 256 registers that two waves a SIMD leave each (in registers, 21
    // words were spilled, prefetched tiles among them: 1115 us for both passes over 2 x 16 heads of 4096 x 4096 instead of 1005)
    constexpr bool VLDS = sizeof(T) == 2 && DP == 128;
    __shared__ __attribute__((aligned(16))) char lds[4 * TB + (VLDS ? 4 * TV : 0)];
    __shared__ __attribute__((aligned(16))) float stat[2][2][RT];       // lse (units of log2) and delta of a tile's rows
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
    const int Hq = p.Hk * p.G, tiles = (p.Tk + 127) / 128;
    int lin = on_xcd(p, blockIdx.x, tiles * p.B * p.Hk * p.nsplit * (BOTH ? 1 : 2));
    const bool want_dk = !BOTH && (lin & 1);                              // !BOTH: this workgroup's job
    if (!BOTH) lin >>= 1;
    const int split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int key = w.tile * 128 + wave * 32 + col;
    const int first = w.tile * 128 + wave * 32;
    const bool ok = (key_bits(key_byte(p, w, first, w.klen, lane), first, w.klen, lane) >> col) & 1;
    const float c = p.scale * LOG2E;

    const int rows = w.tile * 128 < w.klen ? w.qlen * p.G : 0;
    const Span span = split_span(rows, RT, p.nsplit, split, true);
    const int rbeg = span.beg, rend = span.end;
    const int nt = rend > rbeg ? (rend - rbeg + RT - 1) / RT : 0;
    Stage<T, DP, RT, 256> sq, so;
    float lse2 = INFINITY, delta = 0.f;
    // where the group divides the rows that a thread's pieces lie apart, those and the next tile's are the same heads at later steps
    const bool even = sq.STEP % p.G == 0;
    const int64_t qstep = sq.STEP / p.G * p.qs[1], ostep = sq.STEP / p.G * p.ds[1];
    const int r1 = rbeg + tid / sq.CPR, d1 = tid % sq.CPR * sq.PER < p.D ? tid % sq.CPR * sq.PER : 0;
    const T* q1 = row_ptr<T>(p, p.q, w, r1, p.qs[0], p.qs[1], p.qs[2]) + d1;
    const T* o1 = row_ptr<T>(p, p.dout, w, r1, p.ds[0], p.ds[1], p.ds[2]) + d1;
    auto fetch = [&](int j) {
        const int r0 = rbeg + j * RT;
        if (even && r0 + RT <= rend) {
#pragma unroll
            for (int i = 0; i < sq.N; ++i) {
                sq.x[i] = load16(q1);
                so.x[i] = load16(o1);
                q1 += qstep;
                o1 += ostep;
            }
        } else {
            sq.load([&](int i) { return row_ptr<T>(p, p.q, w, r0 + i, p.qs[0], p.qs[1], p.qs[2]); }, p.D, tid);
            so.load([&](int i) { return row_ptr<T>(p, p.dout, w, r0 + i, p.ds[0], p.ds[1], p.ds[2]); }, p.D, tid);
        }
        if (tid < RT) {
            const int r = r0 + tid, t = row_time(p, r);
            lse2 = INFINITY;
            delta = 0.f;
            if (r < rend) {
                const int64_t at = ((int64_t)w.b * Hq + w.hk * p.G + r - t * p.G) * p.Tq + t;
                const float lse = p.lse[at];
                if (lse != -INFINITY) lse2 = lse * LOG2E;
                delta = p.aux[at];
            }
        }
    };
    auto commit = [&](int j) {
        char* x = lds + (j & 1) * 2 * TB;
        const int left = rend - (rbeg + j * RT);
        const uint64_t bits = left >= RT ? (RT == 64 ? ~0ull : 0xffffffffull) : (1ull << left) - 1;
        sq.store(x, bits, p.D, tid);
        so.store(x + TB, bits, p.D, tid);
        if (tid < RT) { stat[j & 1][0][tid] = lse2; stat[j & 1][1][tid] = delta; }
    };
    if (nt) fetch(0);                                    // on its way while the keys' operands are loaded

    frag_t<T> K[DP / 16], V[DP / 16];
    f32x16 acc[NACC][DP / 32];                                            // dv first
    const int64_t kk = min(key, p.Tk - 1);
    row_frags<T, DP>(K, (const T*)p.k + w.b * p.ks[0] + w.hk * p.ks[2] + kk * p.ks[1], p.D, ok, half);
    char* tv = lds + 4 * TB + wave * TV;
    float by = 1.f;
    if (BOTH || want_dk) {
        row_frags<T, DP>(V, (const T*)p.v + w.b * p.vs[0] + w.hk * p.vs[2] + kk * p.vs[1], p.D, ok, half);
        if constexpr (__is_same(T, f16_t)) {
            float n = 0.f, d = 0.f;
            const int parts = rows ? (p.Tq * p.G + 127) / 128 : 0;
            const float* from = range_of<T>(p, w, parts);
            for (int i = lane; i < parts * 4; i += 64) {
                n = fmaxf(n, from[2 * i]);
                d = fmaxf(d, from[2 * i + 1]);
            }
            const float most = wave_max(n) * norm_of<T>(V) + wave_max(d);
            if (most > 32768.f && most < INFINITY) by = ldexpf(1.f, 14 - ilogbf(most));
        }
        if constexpr (VLDS) {
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) *(frag_t<T>*)(tv + col * Tile<T, DP>::STRIDE + (s * 16 + half * 8) * 2) = V[s];
            wave_lds_fence();
        }
    }
#pragma unroll
    for (int a = 0; a < NACC; ++a)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[a][d] = f32x16{};

    if (nt) commit(0);
    for (int j = 0; j < nt; ++j) {
        __syncthreads();
        if (j + 1 < nt) fetch(j + 1);
        const char *tq = lds + (j & 1) * 2 * TB, *to = tq + TB;
#pragma unroll
        for (int q0 = 0; q0 < RT; q0 += 32) {
            f32x16 S = {};
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) S = El<T>::mma(row_frag<T, DP>(tq, q0, s, lane), K[s], S);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 l = *(const f32x4*)&stat[j & 1][0][q0 + 8 * g + 4 * half];
#pragma unroll
                for (int i = 0; i < 4; ++i) S[4 * g + i] = exp2_(fmaf(S[4 * g + i], c, -l[i]));
            }
            if (BOTH || !want_dk) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const frag_t<T> P = next_frag<T>(S, s);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) acc[0][d] = El<T>::mma(trans_frag<T, DP>(to, q0 + 16 * s, 32 * d, lane), P, acc[0][d]);
                }
            }
            if (BOTH || want_dk) {
                f32x16 dP = {};
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) dP = El<T>::mma(row_frag<T, DP>(to, q0, s, lane), VLDS ? row_frag<T, DP>(tv, 0, s, lane) : V[s], dP);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = *(const f32x4*)&stat[j & 1][1][q0 + 8 * g + 4 * half];
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[4 * g + i] *= __is_same(T, f16_t) ? (dP[4 * g + i] - x[i]) * by : dP[4 * g + i] - x[i];
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const frag_t<T> dS = next_frag<T>(S, s);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d)
                        acc[NACC - 1][d] = El<T>::mma(trans_frag<T, DP>(tq, q0 + 16 * s, 32 * d, lane), dS, acc[NACC - 1][d]);
                }
            }
        }
        if (j + 1 < nt) commit(j + 1);
    }

    if (key < p.Tk) {
        const int64_t n = (int64_t)p.B * p.Tk * p.Hk * p.D, at = (((int64_t)w.b * p.Tk + key) * p.Hk + w.hk) * p.D;
#pragma unroll
        for (int a = 0; a < NACC; ++a) {
            const bool dk = BOTH ? a == 1 : want_dk;
            T* o = (T*)(dk ? p.o1 : p.o0) + at;
            float* part = p.part + ((dk ? p.nsplit : 0) + split) * n + at;
            const float f = dk ? p.scale / by : 1.f;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int e = 32 * d + 8 * g + 4 * half;
                    f32x4 x = {acc[a][d][4 * g], acc[a][d][4 * g + 1], acc[a][d][4 * g + 2], acc[a][d][4 * g + 3]};
                    x = ok ? x * f : f32x4{0.f, 0.f, 0.f, 0.f};
                    if (e < p.D) {
                        if (p.nsplit == 1) store4<T>(o + e, x);
                        else *(f32x4*)(part + e) = x;
                    }
                }
        }
    }
}

// out[i] = the sum of the splits' results in their order; y = 1: dk
struct SumP { const float* part; void *o0, *o1; int64_t n; int nsplit; };
template <class T> __global__ __launch_bounds__(256) void attn_sum(const SumP p) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= p.n) return;                                                 // n is a multiple of 8
    const float* at = p.part + blockIdx.y * p.nsplit * p.n + i;
    f32x4 s = *(const f32x4*)at;
    for (int k = 1; k < p.nsplit; ++k) s += *(const f32x4*)(at + k * p.n);
    store4<T>((T*)(blockIdx.y ? p.o1 : p.o0) + i, s);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------
struct GradPlan { bool small; int dq_split, kv_split; int64_t dq_units, kv_units, nq, nk; };
static int split_for(int64_t units, int64_t pieces, int64_t groups) {
    const int64_t n = units > 0 ? groups / units : 1, k = n < pieces ? n : pieces;
    return (int)(k < 1 ? 1 : k > 16 ? 16 : k);
}
static GradPlan gradient_plan(const oph_seq_attn* a) {
    const int64_t M = (int64_t)a->Tq * (a->Hq / a->Hk), heads = (int64_t)a->B * a->Hk;
    GradPlan g;
    // fp32 on 16x16 products: where 128 x 128 tiles are too few to fill the machine and too few scores lie in them (16 sequences of 200 x 150:
    // x 64 22 us, 63 on the large tiles, x 128 36 and 110; two heads of that x 128 70 and 111; but 4 x 4 heads of 100 x 1500 x 64 68 and 56,
    // 64 x 8 heads of 30 x 30 x 64 34 and 28), and for D > 128, where the large tiles' operands do not fit the registers (4 x 8 heads of
    // 1024 x 1024 x 256: 1490 and 2817).
    g.small = a->dtype == OPH_SEQ_F32 &&
              (a->D > 128 || (cdiv(M, 128) * heads * cdiv(a->Tk, 128) < 256 && M * heads * a->Tk < (a->D <= 64 ? 2300000 : 1600000)));
    const int rows = g.small ? 16 : 128, keys = g.small ? 16 : 128;
    g.dq_units = cdiv(M, rows) * heads;
    g.kv_units = cdiv(a->Tk, keys) * heads * (g.small || a->D <= 128 ? 1 : 2);
    // 512 workgroups, 256 for D > 128: one round of two or one a CU; two rounds of attn16_dkv and of fp32 above D = 64, one of which fills a CU's
    // registers.  At least 128 keys or rows a split (16 x 200 x 150 x 128 fp32: 36 us whole, 54 in two splits)
    const int64_t groups = a->D > 128 ? 256 : 512;
    g.dq_split = split_for(g.dq_units, a->Tk / 128, groups);
    g.kv_split = split_for(g.kv_units, M / 128, groups);
    g.nq = (int64_t)a->B * a->Tq * a->Hq * a->D;
    g.nk = (int64_t)a->B * a->Tk * a->Hk * a->D;
    return g;
}
// delta, and for float16 the largest |dout| and |delta| of every 32 rows (range_of())
static int64_t delta_floats(const oph_seq_attn* a) {
    const int64_t G = a->Hq / a->Hk, range = a->dtype == OPH_SEQ_F16 ? cdiv(a->Tq * G, 128) * 8 * a->B * a->Hk : 0;
    return cdiv((int64_t)a->B * a->Hq * a->Tq, 4) * 4 + range;
}
int64_t attn_gradient_workspace(const oph_seq_attn* a) {
    const GradPlan g = gradient_plan(a);
    const int64_t q = g.dq_split > 1 ? g.dq_split * g.nq : 0, k = g.kv_split > 1 ? 2 * g.kv_split * g.nk : 0;
    return (delta_floats(a) + (q > k ? q : k)) * (int64_t)sizeof(float);   // the two passes use the same partial results' space in turn
}

template <class T> static int sum(const float* part, void* o0, void* o1, int64_t n, int nsplit, void* stream) {
    const SumP s = {part, o0, o1, n, nsplit};
    return launch<SumP>(attn_sum<T>, dim3((unsigned)cdiv(n, 1024), o1 ? 2 : 1), 256, s, 0, stream);
}
template <class T, int DP> static int gradient(const oph_seq_attn* a, AttnP p, void* stream) {
    const GradPlan g = gradient_plan(a);
    if (g.nq) {
        p.nsplit = g.dq_split;
        p.o0 = a->dq;
        const int64_t groups = g.dq_units * g.dq_split;
        p.chunk = run_of(a, groups, false);
        int rc;
        if constexpr (sizeof(T) == 4 && DP > 128) rc = attn16_launch(p, groups, 1, stream);
        else rc = g.small ? attn16_launch(p, groups, 1, stream) : launch<AttnP>(attn_dq<T, DP>, dim3((unsigned)groups), 256, p, 0, stream);
        if (rc) return rc;
        if (g.dq_split > 1) {
            if (int rc = sum<T>(p.part, a->dq, nullptr, g.nq, g.dq_split, stream)) return rc;
        }
    }
    if (g.nk) {
        p.nsplit = g.kv_split;
        p.o0 = a->dv;
        p.o1 = a->dk;
        const int64_t groups = g.kv_units * g.kv_split;
        p.chunk = run_of(a, groups, false);
        int rc;
        if constexpr (sizeof(T) == 4 && DP > 128) rc = attn16_launch(p, groups, 2, stream);
        else rc = g.small ? attn16_launch(p, groups, 2, stream) : launch<AttnP>(attn_dkv<T, DP, DP <= 128>, dim3((unsigned)groups), 256, p, 0, stream);
        if (rc) return rc;
        if (g.kv_split > 1) return sum<T>(p.part, a->dv, a->dk, g.nk, g.kv_split, stream);
    }
    return OPH_OK;
}
template <class T> static int gradient_d(const oph_seq_attn* a, const AttnP& p, void* stream) {
    if (p.D <= 64) return gradient<T, 64>(a, p, stream);
    if (p.D <= 128) return gradient<T, 128>(a, p, stream);
    return gradient<T, 256>(a, p, stream);
}

}  // namespace ophseq

using namespace ophseq;
extern "C" int oph_seq_attn_gradient(const oph_seq_attn* a, int device, void* stream) {
    if (int rc = attn_check(a, true)) return rc;
    if (!a->B || (!a->Tq && !a->Tk)) return OPH_OK;
    if (a->Tq && (!a->q || !a->out || !a->lse || !a->dout || !a->dq)) return fail(OPH_ERR_INVALID, "attention: q, out, lse, dout and dq must not be NULL");
    if (a->Tk && (!a->k || !a->v || !a->dk || !a->dv)) return fail(OPH_ERR_INVALID, "attention: k, v, dk and dv must not be NULL");
    const int64_t need = attn_gradient_workspace(a);
    if (need && (!a->workspace || (int64_t)a->workspace_bytes < need || ((uintptr_t)a->workspace & 15)))
        return fail(OPH_ERR_INVALID, "attention: the workspace must hold %lld bytes, 16-byte aligned", (long long)need);
    OnDevice on(device);
    if (on.status) return on.status;
    AttnP p = attn_params(a);
    p.out = a->out;
    p.dout = a->dout;
    p.lse = a->lse;
    p.aux = (float*)a->workspace;
    p.part = p.aux + delta_floats(a);
    for (int i = 0; i < 3; ++i) p.ds[i] = a->dout_stride[i];
    if (a->dtype == OPH_SEQ_F32) return gradient_d<float>(a, p, stream);
    if (a->dtype == OPH_SEQ_BF16) return gradient_d<bf16_t>(a, p, stream);
    return gradient_d<f16_t>(a, p, stream);
}
