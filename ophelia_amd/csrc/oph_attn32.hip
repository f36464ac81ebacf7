// Cross attention in fp32 for problems that do not fill the machine with 128-row workgroups: forward and gradient on 16x16x4 products.
//
// The fp32 matrix rate is a sixteenth of the 16-bit one, so a tile's time is its products' and not its loads': operands come straight from
// memory (row pieces of 64 bytes, columns of 64 bytes), no tile is shared through LDS.  A workgroup owns 16 rows (forward, dq) or 16
// keys (dk, dv) and its 4 waves take every fourth tile of 16 of the other axis; their results meet in LDS in the order of the waves.
// 16 instead of 32 rows halve both the work of a partly filled tile and the registers of D = 256: all operands and results of a
// tile are resident (forward 4, dq 5, dk + dv 6 times 64 registers).
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

// a row's operand: elements 16s + 4(l/16) .. + 3, zeros where !ok and beyond D
template <int DP> __device__ __forceinline__ void rows16(f32x4 (&f)[DP / 16], const float* row, int D, bool ok, int g) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = 16 * s + 4 * g;
        const f32x4 x = loadf4(row + (d < D ? d : 0));
        f[s] = ok && d < D ? x : f32x4{0.f, 0.f, 0.f, 0.f};
    }
}
// the transposed operand: element j is column 16s + l%16 of the row that ptr[j] points to
template <int DP> __device__ __forceinline__ void cols16(f32x4 (&f)[DP / 16], const float* const (&ptr)[4], int D, int col) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = 16 * s + col < D ? 16 * s + col : 0;              // columns beyond D are results that nobody stores
#pragma unroll
        for (int j = 0; j < 4; ++j) f[s][j] = ptr[j][d];
    }
}
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

// results (columns of 16 x D of the four waves) -> row-major in LDS -> sums of the waves, four columns of D at a time to `out(row, d, sum)`
template <int DP, class F> __device__ __forceinline__ void meet16(float* lds, const f32x4 (&x)[DP / 16], float weight, F out) {
    constexpr int LD = DP + 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) *(f32x4*)(lds + (wave * 16 + col) * LD + 16 * s + 4 * g) = x[s] * weight;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        const int c = i * 256 + tid, row = c / (DP / 4), d = c % (DP / 4) * 4;
        f32x4 sum = *(const f32x4*)(lds + row * LD + d);
#pragma unroll
        for (int w = 1; w < 4; ++w) sum += *(const f32x4*)(lds + (w * 16 + row) * LD + d);
        out(row, d, sum);
    }
}

template <int DP> __global__ __launch_bounds__(256) void attn16_forward(const AttnP p) {
    __shared__ __attribute__((aligned(16))) float lds[64 * (DP + 4)];
    __shared__ float ml[4][16][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int M = p.Tq * p.G, tiles = (M + 15) / 16;
    const int lin = on_xcd(blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int row0 = w.tile * 16;
    const float c = p.scale * LOG2E;
    const int per = ((w.klen + 15) / 16 + p.nsplit - 1) / p.nsplit * 16;
    const int kbeg = split * per, kend = row_time(p, row0) < w.qlen ? min(w.klen, kbeg + per) : kbeg;
    f32x4 Q[DP / 16], O[DP / 16];
    {
        const int r = row0 + col;
        rows16<DP>(Q, row_ptr<float>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]), p.D, r < M && row_time(p, r) < w.qlen, g);
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) O[s] = f32x4{};
    float m = -INFINITY, l = 0.f;
    const float* k = (const float*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const float* v = (const float*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    for (int key0 = kbeg + wave * 16; key0 < kend; key0 += 64) {
        const uint32_t bits = (uint32_t)key_bits(p, w, key0, kend, lane) & 0xffffu;
        if (!bits) continue;
        f32x4 K[DP / 16], V[DP / 16], S = {};
        rows16<DP>(K, k + (int64_t)min(key0 + col, kend - 1) * p.ks[1], p.D, true, g);
        const float* at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = v + (int64_t)min(key0 + 4 * g + j, kend - 1) * p.vs[1];
        cols16<DP>(V, at, p.D, col);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S = mma16(K[s], Q[s], S);
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
        if (bits != 0xffffu) keep16(V, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) O[s] = mma16(V[s], S, O[s]);
    }
    l = over_groups(l, false);
    if (g == 0) { ml[wave][col][0] = m; ml[wave][col][1] = l; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i][col][0]);
    const int64_t unit = ((int64_t)(w.b * p.Hk + w.hk) * tiles + w.tile) * p.nsplit + split;
    meet16<DP>(lds, O, exp2_(m - (top == -INFINITY ? 0.f : top)), [&](int row, int d, f32x4 o) {
        const int r = row0 + row, t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
        if (r >= M || d >= p.D) return;
        float om = -INFINITY, ol = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) om = fmaxf(om, ml[i][row][0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) ol += ml[i][row][1] * exp2_(ml[i][row][0] - (om == -INFINITY ? 0.f : om));
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

template <int DP> __global__ __launch_bounds__(256) void attn16_dq(const AttnP p) {
    __shared__ __attribute__((aligned(16))) float lds[64 * (DP + 4)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int M = p.Tq * p.G, Hq = p.Hk * p.G, tiles = (M + 15) / 16;
    const int lin = on_xcd(blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int row0 = w.tile * 16, r = row0 + col, t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
    const bool row = r < M && t < w.qlen;
    const float c = p.scale * LOG2E;
    const int per = ((w.klen + 15) / 16 + p.nsplit - 1) / p.nsplit * 16;
    const int kbeg = split * per, kend = row_time(p, row0) < w.qlen ? min(w.klen, kbeg + per) : kbeg;
    f32x4 Q[DP / 16], dO[DP / 16], dQ[DP / 16];
    rows16<DP>(Q, row_ptr<float>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]), p.D, row, g);
    rows16<DP>(dO, row_ptr<float>(p, p.dout, w, r, p.ds[0], p.ds[1], p.ds[2]), p.D, row, g);
    float delta = 0.f, lse2 = INFINITY;
    {
        rows16<DP>(dQ, row_ptr<float>(p, p.out, w, r, (int64_t)p.Tq * Hq * p.D, (int64_t)Hq * p.D, p.D), p.D, row, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) delta = fmaf(dQ[s][j], dO[s][j], delta);
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
    const float* k = (const float*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const float* v = (const float*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    for (int key0 = kbeg + wave * 16; key0 < kend; key0 += 64) {
        const uint32_t bits = (uint32_t)key_bits(p, w, key0, kend, lane) & 0xffffu;
        if (!bits) continue;
        f32x4 K[DP / 16], V[DP / 16], S = {}, dP = {};
        const int64_t mine = min(key0 + col, kend - 1);
        rows16<DP>(K, k + mine * p.ks[1], p.D, true, g);
        rows16<DP>(V, v + mine * p.vs[1], p.D, true, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S = mma16(K[s], Q[s], S);
        const float* at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = k + (int64_t)min(key0 + 4 * g + j, kend - 1) * p.ks[1];
        cols16<DP>(K, at, p.D, col);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dP = mma16(V[s], dO[s], dP);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[j] = (bits >> (4 * g + j)) & 1 ? exp2_(fmaf(S[j], c, -lse2)) * (dP[j] - delta) : 0.f;
        if (bits != 0xffffu) keep16(K, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dQ[s] = mma16(K[s], S, dQ[s]);
    }
    meet16<DP>(lds, dQ, p.scale, [&](int i, int d, f32x4 x) {
        const int rr = row0 + i, tt = row_time(p, rr), hh = w.hk * p.G + rr - tt * p.G;
        if (rr >= M || d >= p.D) return;
        const int64_t at = (((int64_t)w.b * p.Tq + tt) * Hq + hh) * p.D + d;
        if (tt >= w.qlen) x = f32x4{0.f, 0.f, 0.f, 0.f};
        float* o = p.nsplit == 1 ? (float*)p.o0 : p.part + (int64_t)split * p.B * p.Tq * Hq * p.D;
        store4<float>(o + at, x);
    });
}

template <int DP> __global__ __launch_bounds__(256) void attn16_dkv(const AttnP p) {
    __shared__ __attribute__((aligned(16))) float lds[64 * (DP + 4)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int Hq = p.Hk * p.G, tiles = (p.Tk + 15) / 16;
    const int lin = on_xcd(blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int key0 = w.tile * 16;
    const uint32_t keys = (uint32_t)key_bits(p, w, key0, w.klen, lane) & 0xffffu;
    const float c = p.scale * LOG2E;
    f32x4 K[DP / 16], V[DP / 16], dK[DP / 16], dV[DP / 16];
    {
        const int64_t key = min(key0 + col, p.Tk - 1);
        const bool ok = (keys >> col) & 1;
        rows16<DP>(K, (const float*)p.k + w.b * p.ks[0] + w.hk * p.ks[2] + key * p.ks[1], p.D, ok, g);
        rows16<DP>(V, (const float*)p.v + w.b * p.vs[0] + w.hk * p.vs[2] + key * p.vs[1], p.D, ok, g);
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) dK[s] = dV[s] = f32x4{};
    const int rows = keys ? w.qlen * p.G : 0;
    const int per = ((rows + 15) / 16 + p.nsplit - 1) / p.nsplit * 16;
    const int rbeg = split * per, rend = min(rows, rbeg + per);
    for (int r0 = rbeg + wave * 16; r0 < rend; r0 += 64) {
        const uint32_t bits = rend - r0 >= 16 ? 0xffffu : (1u << (rend - r0)) - 1;
        f32x4 X[DP / 16], S = {}, dP = {};
        float lse2[4], delta[4];
        const float *qa[4], *oa[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = min(r0 + 4 * g + j, rend - 1), t = row_time(p, r);
            qa[j] = row_ptr<float>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]);
            oa[j] = row_ptr<float>(p, p.dout, w, r, p.ds[0], p.ds[1], p.ds[2]);
            const int64_t at = ((int64_t)w.b * Hq + w.hk * p.G + r - t * p.G) * p.Tq + t;
            lse2[j] = p.lse[at];
            lse2[j] = lse2[j] == -INFINITY ? INFINITY : lse2[j] * LOG2E;
            delta[j] = p.aux[at];
        }
        const int mine = min(r0 + col, rend - 1);
        rows16<DP>(X, row_ptr<float>(p, p.q, w, mine, p.qs[0], p.qs[1], p.qs[2]), p.D, true, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S = mma16(X[s], K[s], S);
        rows16<DP>(X, row_ptr<float>(p, p.dout, w, mine, p.ds[0], p.ds[1], p.ds[2]), p.D, true, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dP = mma16(X[s], V[s], dP);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[j] = (bits >> (4 * g + j)) & 1 ? exp2_(fmaf(S[j], c, -lse2[j])) : 0.f;
        cols16<DP>(X, oa, p.D, col);
        if (bits != 0xffffu) keep16(X, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dV[s] = mma16(X[s], S, dV[s]);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[j] = (bits >> (4 * g + j)) & 1 ? S[j] * (dP[j] - delta[j]) : 0.f;
        cols16<DP>(X, qa, p.D, col);
        if (bits != 0xffffu) keep16(X, bits, g);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) dK[s] = mma16(X[s], S, dK[s]);
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
    meet16<DP>(lds, dV, 1.f, [&](int i, int d, f32x4 x) { store(i, d, x, false); });
    __syncthreads();
    meet16<DP>(lds, dK, p.scale, [&](int i, int d, f32x4 x) { store(i, d, x, true); });
}

template <int DP> static int go(const AttnP& p, int64_t groups, int what, void* stream) {
    return launch<AttnP>(what == 0 ? attn16_forward<DP> : what == 1 ? attn16_dq<DP> : attn16_dkv<DP>, dim3((unsigned)groups), 256, p, 0, stream);
}
int attn16_launch(const AttnP& p, int64_t groups, int what, void* stream) {
    return p.D <= 64 ? go<64>(p, groups, what, stream) : p.D <= 128 ? go<128>(p, groups, what, stream) : go<256>(p, groups, what, stream);
}

}  // namespace ophseq
