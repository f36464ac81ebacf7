// Cross attention in fp32 for problems that do not fill the machine with 128-row workgroups: forward and gradient on 16x16x4 products.
//
// The fp32 matrix rate is a sixteenth of the 16-bit one, so operands come straight from memory (row pieces of 64 bytes, columns of 64 bytes)
// and no tile of the other axis is shared through LDS.  What bounds them on long inputs is the return of these pieces (4 x 8 heads of 1024 x
// 1024 x 256, gradient with respect to the queries: 660 us, 87 % of them busy with it, the matrix units half of the time); on short ones,
// which they are for, latency.  A workgroup owns 16 rows
// (forward, dq) or 16 keys (dk, dv), whose operands its NW waves share in LDS; every wave takes every NW-th tile of 16 of the other axis, and
// their results are added in a fixed order at the end.  16 instead of 32 rows halve both the work of a partly filled tile and the
// registers of D = 256: with the shared operands in LDS the waves (4, or 8 where two fit a SIMD) have room for their results and for
// two tiles x and y of what comes from memory: as soon as the products that read one are issued it takes its next load, a product ahead of its next use.
//
// Layout of a 16x16 product: lane l holds column l % 16 and rows 4(l/16) + j in register j; as the operand of the next product register j
// is the element of step j, which contracts rows {j, 4 + j, 8 + j, 12 + j}, and the other operand is read in the same order.
#include "oph_attn.h"

#include <math.h>

namespace ophseq {

__device__ __forceinline__ f32x4 mma16(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 loadf4(const float* p) { return __builtin_bit_cast(f32x4, load16(p)); }

// A row's operand: elements 16s + 4(l/16) .. + 3.  EXACT: D == DP; otherwise what lies beyond D is not the row's, and edge16() clears it
// before its use.
template <int DP, bool EXACT> __device__ __forceinline__ void rows16(f32x4 (&f)[DP / 16], const float* row, int D, int g) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) f[s] = loadf4(row + (EXACT || 16 * s + 4 * g < D ? 16 * s + 4 * g : 0));
}
template <int DP, bool EXACT> __device__ __forceinline__ void edge16(f32x4 (&f)[DP / 16], int D, int g) {
    if (!EXACT)
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) f[s] = 16 * s + 4 * g < D ? f[s] : f32x4{0.f, 0.f, 0.f, 0.f};
}
// 16 rows shared in LDS as operands: cleared where !ok and beyond D
template <int DP, int NW, class F> __device__ __forceinline__ void share16(float* tile, F row, uint32_t bits, int D) {
#pragma unroll
    for (int i = 0; i < (16 * (DP / 4) + 64 * NW - 1) / (64 * NW); ++i) {
        const int c = i * 64 * NW + threadIdx.x, r = c / (DP / 4), d = c % (DP / 4) * 4;
        if (16 * (DP / 4) % (64 * NW) && r >= 16) break;
        const f32x4 x = loadf4(row(r) + (d < D ? d : 0));
        *(f32x4*)(tile + r * (DP + 4) + d) = d < D && ((bits >> r) & 1) ? x : f32x4{0.f, 0.f, 0.f, 0.f};
    }
}
template <int DP> __device__ __forceinline__ f32x4 shared16(const float* tile, int s, int col, int g) {
    return *(const f32x4*)(tile + col * (DP + 4) + 16 * s + 4 * g);
}
// the transposed operand: element j is column 16s + l%16 of the row that ptr[j] points to; columns beyond D are results that nobody stores
template <int DP, bool EXACT> __device__ __forceinline__ void cols16(f32x4 (&f)[DP / 16], const float* const (&ptr)[4], int D, int col) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[s][j] = ptr[j][EXACT || 16 * s + col < D ? 16 * s + col : 0];
}
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 16 ? 0xffffu : n > 0 ? (1u << n) - 1 : 0; }
template <int N> __device__ __forceinline__ void keep16(f32x4 (&f)[N], uint32_t bits, int g) {      // rows without their bit may be NaN
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[s][j] = (bits >> (4 * g + j)) & 1 ? f[s][j] : 0.f;
}
__device__ __forceinline__ float over_groups(float x, bool max) {       // over the four lanes of a column
#pragma unroll
    for (int i = 16; i < 64; i <<= 1) {
        const float y = __shfl_xor(x, i);
        x = max ? fmaxf(x, y) : x + y;
    }
    return x;
}

// results (columns of 16 x D of the waves) -> sums, four columns of D at a time to `out(row, d, sum)`: waves 4..7, if there, are added to 0..3
// first, then those in their order.  All waves are past their last use of `lds`.
template <int DP, int NW, class F> __device__ __forceinline__ void meet16(float* lds, f32x4 (&x)[DP / 16], float weight, F out) {
    constexpr int LD = DP + 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    float* at = lds + ((wave & 3) * 16 + col) * LD + 4 * g;
    if (NW == 8) {
        if (wave >= 4)
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) *(f32x4*)(at + 16 * s) = x[s] * weight;
        __syncthreads();
        if (wave < 4)
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) *(f32x4*)(at + 16 * s) = x[s] * weight + *(const f32x4*)(at + 16 * s);
    } else {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) *(f32x4*)(at + 16 * s) = x[s] * weight;
    }
    __syncthreads();
    for (int c = tid; c < 16 * (DP / 4); c += 64 * NW) {
        const int row = c / (DP / 4), d = c % (DP / 4) * 4;
        f32x4 sum = *(const f32x4*)(lds + row * LD + d);
#pragma unroll
        for (int w = 1; w < 4; ++w) sum += *(const f32x4*)(lds + (w * 16 + row) * LD + d);
        out(row, d, sum);
    }
}

template <int DP, bool EXACT, int NW> __global__ __launch_bounds__(64 * NW) void attn16_forward(const AttnP p) {
    __shared__ __attribute__((aligned(16))) float lds[64 * (DP + 4)];
    __shared__ float ml[NW][16][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int M = p.Tq * p.G, tiles = (M + 15) / 16;
    const int lin = on_xcd(p, blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int row0 = w.tile * 16;
    const float c = p.scale * LOG2E;
    const Span span = split_span(w.klen, 16, p.nsplit, split, row_time(p, row0) < w.qlen);
    const int kbeg = span.beg, kend = span.end;
    const float* k = (const float*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const float* v = (const float*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    f32x4 O[DP / 16], x[DP / 16], y[DP / 16];                            // x: rows of keys, y: columns of values
    auto fetch_k = [&](int key0) { rows16<DP, EXACT>(x, k + (int64_t)min(key0 + col, kend - 1) * p.ks[1], p.D, g); };
    auto fetch_v = [&](int key0) {
        const float* at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = v + (int64_t)min(key0 + 4 * g + j, kend - 1) * p.vs[1];
        cols16<DP, EXACT>(y, at, p.D, col);
    };
    int key0 = kbeg + wave * 16;
    uint8_t byte = key_byte(p, w, key0, kend, lane);
    if (key0 < kend) {
        fetch_k(key0);
        fetch_v(key0);
    }
    share16<DP, NW>(lds, [&](int i) { return row_ptr<float>(p, p.q, w, row0 + i, p.qs[0], p.qs[1], p.qs[2]); }, bits_below(min(M, w.qlen * p.G) - row0), p.D);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) O[s] = f32x4{};
    float m = -INFINITY, l = 0.f;
    for (; key0 < kend; key0 += 16 * NW) {
        const uint32_t bits = (uint32_t)key_bits(byte, key0, kend, lane) & 0xffffu;
        f32x4 S = {};
        edge16<DP, EXACT>(x, p.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S = mma16(x[s], shared16<DP>(lds, s, col, g), S);
        if (key0 + 16 * NW < kend) {
            byte = key_byte(p, w, key0 + 16 * NW, kend, lane);
            fetch_k(key0 + 16 * NW);
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            S[j] = (bits >> (4 * g + j)) & 1 ? S[j] : -INFINITY;
            top = fmaxf(top, S[j]);
        }
        top = fmaxf(m, over_groups(top, true) * c);
        const float base = top == -INFINITY ? 0.f : top, shrink = exp2_(m - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            S[j] = exp2_(fmaf(S[j], c, -base));
            sum += S[j];
        }
        l = l * shrink + sum;
        m = top;
        if (__any(shrink != 1.f)) {
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) O[s] *= shrink;
        }
        if (bits != 0xffffu) keep16(y, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) O[s] = mma16(y[s], S, O[s]);
        if (key0 + 16 * NW < kend) fetch_v(key0 + 16 * NW);
    }
    l = over_groups(l, false);
    if (g == 0) { ml[wave][col][0] = m; ml[wave][col][1] = l; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, ml[i][col][0]);
    const int64_t unit = ((int64_t)(w.b * p.Hk + w.hk) * tiles + w.tile) * p.nsplit + split;
    meet16<DP, NW>(lds, O, exp2_(m - (top == -INFINITY ? 0.f : top)), [&](int row, int d, f32x4 o) {
        const int r = row0 + row, t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
        if (r >= M || d >= p.D) return;
        float om = -INFINITY, ol = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) om = fmaxf(om, ml[i][row][0]);
#pragma unroll
        for (int i = 0; i < NW; ++i) ol += ml[i][row][1] * exp2_(ml[i][row][0] - (om == -INFINITY ? 0.f : om));
        if (p.nsplit == 1) {
            const bool live = t < w.qlen && ol != 0.f;
            store4<float>((float*)p.o0 + (((int64_t)w.b * p.Tq + t) * (p.Hk * p.G) + h) * p.D + d, live ? o * (1.f / ol) : f32x4{0.f, 0.f, 0.f, 0.f});
            if (d == 0) p.lse[((int64_t)w.b * (p.Hk * p.G) + h) * p.Tq + t] = live ? (om + log2f(ol)) * LN2 : -INFINITY;
        } else {
            *(f32x4*)(p.part + (unit * 16 + row) * DP + d) = o;
            if (d == 0) { p.aux[(unit * 16 + row) * 2] = om; p.aux[(unit * 16 + row) * 2 + 1] = ol; }
        }
    });
}

template <int DP, bool EXACT, int NW> __global__ __launch_bounds__(64 * NW) void attn16_dq(const AttnP p) {
    __shared__ __attribute__((aligned(16))) float lds[64 * (DP + 4)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int M = p.Tq * p.G, Hq = p.Hk * p.G, tiles = (M + 15) / 16;
    const int lin = on_xcd(p, blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int row0 = w.tile * 16, r = row0 + col, t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
    const bool row = r < M && t < w.qlen;
    const float c = p.scale * LOG2E;
    const Span span = split_span(w.klen, 16, p.nsplit, split, row_time(p, row0) < w.qlen);
    const int kbeg = span.beg, kend = span.end;
    const float* k = (const float*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const float* v = (const float*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    f32x4 dQ[DP / 16], x[DP / 16], y[DP / 16];                           // x: rows, then columns of keys, y: rows of values
    float *tq = lds, *to = lds + 16 * (DP + 4);
    auto fetch = [&](f32x4 (&f)[DP / 16], const float* base, int64_t stride, int key0) {
        rows16<DP, EXACT>(f, base + (int64_t)min(key0 + col, kend - 1) * stride, p.D, g);
    };
    int key0 = kbeg + wave * 16;
    uint8_t byte = key_byte(p, w, key0, kend, lane);
    if (key0 < kend) {
        fetch(x, k, p.ks[1], key0);
        fetch(y, v, p.vs[1], key0);
    }
    const uint32_t mine = bits_below(min(M, w.qlen * p.G) - row0);
    share16<DP, NW>(tq, [&](int i) { return row_ptr<float>(p, p.q, w, row0 + i, p.qs[0], p.qs[1], p.qs[2]); }, mine, p.D);
    share16<DP, NW>(to, [&](int i) { return row_ptr<float>(p, p.dout, w, row0 + i, p.ds[0], p.ds[1], p.ds[2]); }, mine, p.D);
    rows16<DP, EXACT>(dQ, row_ptr<float>(p, p.out, w, r, (int64_t)p.Tq * Hq * p.D, (int64_t)Hq * p.D, p.D), p.D, g);
    __syncthreads();
    float delta = 0.f, lse2 = INFINITY;
    {
        edge16<DP, EXACT>(dQ, p.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const f32x4 d = shared16<DP>(to, s, col, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) delta = fmaf(dQ[s][j], d[j], delta);
        }
        if (!row) delta = 0.f;
        delta = over_groups(delta, false);
        const int64_t at = ((int64_t)w.b * Hq + h) * p.Tq + t;
        if (row) {
            const float lse = p.lse[at];
            if (lse != -INFINITY) lse2 = lse * LOG2E;
        }
        if (r < M && lane < 16 && wave == 0 && split == 0) p.aux[at] = delta;
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) dQ[s] = f32x4{};
    for (; key0 < kend; key0 += 16 * NW) {
        const uint32_t bits = (uint32_t)key_bits(byte, key0, kend, lane) & 0xffffu;
        f32x4 S = {}, dP = {};
        edge16<DP, EXACT>(x, p.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S = mma16(x[s], shared16<DP>(tq, s, col, g), S);
        const float* at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = k + (int64_t)min(key0 + 4 * g + j, kend - 1) * p.ks[1];
        cols16<DP, EXACT>(x, at, p.D, col);
        edge16<DP, EXACT>(y, p.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dP = mma16(y[s], shared16<DP>(to, s, col, g), dP);
        if (key0 + 16 * NW < kend) {
            byte = key_byte(p, w, key0 + 16 * NW, kend, lane);
            fetch(y, v, p.vs[1], key0 + 16 * NW);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) S[j] = (bits >> (4 * g + j)) & 1 ? exp2_(fmaf(S[j], c, -lse2)) * (dP[j] - delta) : 0.f;
        if (bits != 0xffffu) keep16(x, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dQ[s] = mma16(x[s], S, dQ[s]);
        if (key0 + 16 * NW < kend) fetch(x, k, p.ks[1], key0 + 16 * NW);
    }
    __syncthreads();
    meet16<DP, NW>(lds, dQ, p.scale, [&](int i, int d, f32x4 x) {
        const int rr = row0 + i, tt = row_time(p, rr), hh = w.hk * p.G + rr - tt * p.G;
        if (rr >= M || d >= p.D) return;
        const int64_t at = (((int64_t)w.b * p.Tq + tt) * Hq + hh) * p.D + d;
        if (tt >= w.qlen) x = f32x4{0.f, 0.f, 0.f, 0.f};
        float* o = p.nsplit == 1 ? (float*)p.o0 : p.part + (int64_t)split * p.B * p.Tq * Hq * p.D;
        store4<float>(o + at, x);
    });
}

template <int DP, bool EXACT, int NW> __global__ __launch_bounds__(64 * NW) void attn16_dkv(const AttnP p) {
    __shared__ __attribute__((aligned(16))) float lds[64 * (DP + 4)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int Hq = p.Hk * p.G, tiles = (p.Tk + 15) / 16;
    const int lin = on_xcd(p, blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int key0 = w.tile * 16;
    const uint32_t keys = (uint32_t)key_bits(key_byte(p, w, key0, w.klen, lane), key0, w.klen, lane) & 0xffffu;
    const float c = p.scale * LOG2E;
    const int rows = keys ? w.qlen * p.G : 0;
    const Span span = split_span(rows, 16, p.nsplit, split, true);
    const int rbeg = span.beg, rend = span.end;
    f32x4 dK[DP / 16], dV[DP / 16], x[DP / 16], y[DP / 16];              // x: rows of q, columns of dout, y: rows of dout, columns of q
    float *tk = lds, *tv = lds + 16 * (DP + 4);
    auto q_row = [&](int r) { return row_ptr<float>(p, p.q, w, min(r, rend - 1), p.qs[0], p.qs[1], p.qs[2]); };
    auto o_row = [&](int r) { return row_ptr<float>(p, p.dout, w, min(r, rend - 1), p.ds[0], p.ds[1], p.ds[2]); };
    int r0 = rbeg + wave * 16;
    if (r0 < rend) {
        rows16<DP, EXACT>(x, q_row(r0 + col), p.D, g);
        rows16<DP, EXACT>(y, o_row(r0 + col), p.D, g);
    }
    {
        const float *k = (const float*)p.k + w.b * p.ks[0] + w.hk * p.ks[2], *v = (const float*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
        share16<DP, NW>(tk, [&](int i) { return k + (int64_t)min(key0 + i, p.Tk - 1) * p.ks[1]; }, keys, p.D);
        share16<DP, NW>(tv, [&](int i) { return v + (int64_t)min(key0 + i, p.Tk - 1) * p.vs[1]; }, keys, p.D);
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) dK[s] = dV[s] = f32x4{};
    for (; r0 < rend; r0 += 16 * NW) {
        const uint32_t bits = rend - r0 >= 16 ? 0xffffu : (1u << (rend - r0)) - 1;
        f32x4 S = {}, dP = {};
        float lse2[4], delta[4];
        const float *qa[4], *oa[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = min(r0 + 4 * g + j, rend - 1), t = row_time(p, r);
            qa[j] = q_row(r);
            oa[j] = o_row(r);
            const int64_t at = ((int64_t)w.b * Hq + w.hk * p.G + r - t * p.G) * p.Tq + t;
            lse2[j] = p.lse[at];
            delta[j] = p.aux[at];
        }
        edge16<DP, EXACT>(x, p.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S = mma16(x[s], shared16<DP>(tk, s, col, g), S);
        cols16<DP, EXACT>(x, oa, p.D, col);
        edge16<DP, EXACT>(y, p.D, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dP = mma16(y[s], shared16<DP>(tv, s, col, g), dP);
        cols16<DP, EXACT>(y, qa, p.D, col);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float l = lse2[j] == -INFINITY ? INFINITY : lse2[j] * LOG2E;
            S[j] = (bits >> (4 * g + j)) & 1 ? exp2_(fmaf(S[j], c, -l)) : 0.f;
        }
        if (bits != 0xffffu) keep16(x, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dV[s] = mma16(x[s], S, dV[s]);
        if (r0 + 16 * NW < rend) rows16<DP, EXACT>(x, q_row(r0 + 16 * NW + col), p.D, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[j] = (bits >> (4 * g + j)) & 1 ? S[j] * (dP[j] - delta[j]) : 0.f;
        if (bits != 0xffffu) keep16(y, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dK[s] = mma16(y[s], S, dK[s]);
        if (r0 + 16 * NW < rend) rows16<DP, EXACT>(y, o_row(r0 + 16 * NW + col), p.D, g);
    }
    const int64_t n = (int64_t)p.B * p.Tk * p.Hk * p.D;
    auto store = [&](int i, int d, f32x4 x, bool dk) {
        const int key = key0 + i;
        if (key >= p.Tk || d >= p.D) return;
        const int64_t at = (((int64_t)w.b * p.Tk + key) * p.Hk + w.hk) * p.D + d;
        if (!((keys >> i) & 1)) x = f32x4{0.f, 0.f, 0.f, 0.f};
        float* o = p.nsplit == 1 ? (float*)(dk ? p.o1 : p.o0) : p.part + ((dk ? p.nsplit : 0) + split) * n;
        store4<float>(o + at, x);
    };
    __syncthreads();
    meet16<DP, NW>(lds, dV, 1.f, [&](int i, int d, f32x4 x) { store(i, d, x, false); });
    __syncthreads();
    meet16<DP, NW>(lds, dK, p.scale, [&](int i, int d, f32x4 x) { store(i, d, x, true); });
}

template <int DP, bool EXACT> static int go(const AttnP& p, int64_t groups, int what, void* stream) {
    constexpr int N = DP <= 128 ? 8 : 4, NKV = DP <= 64 ? 8 : 4;          // two waves a SIMD where the registers allow it
    void (*const kernel)(AttnP) = what == 0 ? attn16_forward<DP, EXACT, N> : what == 1 ? attn16_dq<DP, EXACT, N> : attn16_dkv<DP, EXACT, NKV>;
    return launch<AttnP>(kernel, dim3((unsigned)groups), 64 * (what == 2 ? NKV : N), p, 0, stream);
}
template <int DP> static int go_d(const AttnP& p, int64_t groups, int what, void* stream) {
    return p.D == DP ? go<DP, true>(p, groups, what, stream) : go<DP, false>(p, groups, what, stream);
}
int attn16_launch(const AttnP& p, int64_t groups, int what, void* stream) {
    return p.D <= 64 ? go_d<64>(p, groups, what, stream) : p.D <= 128 ? go_d<128>(p, groups, what, stream) : go_d<256>(p, groups, what, stream);
}

}  // namespace ophseq
