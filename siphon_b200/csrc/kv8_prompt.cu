// Attention over the paged 8-bit KV cache for requests with many new tokens
// (prompts and chunks of them), on the tensor cores with accumulators in
// tensor memory.
//
// A CTA owns 256 rows of one KV head (its query heads times consecutive
// tokens) as two tiles of 128, and walks the keys they see 128 at a time:
//   S = Q K^T        tcgen05 MMAs from shared memory, S in tensor memory
//   P = 2^(c S - m)  one thread per row: reads its 128 scores, the running
//                    maximum m (moved only when it grows by 2^8, so the
//                    accumulator is rarely rescaled) and the sum
//   O += P V         P read from tensor memory (over S's columns), O in it
// While one tile's weights are formed, the other's products run. Codes reach
// shared memory as exact f16 (|code| <= 127) written by converter warps in
// the swizzled layout the MMAs read; K's block scales enter with the scores,
// V's with the weights, relative to the largest V scale of the span, so the
// accumulator never changes units.
//
// q enters as two f16 parts (hi + lo; a row of f16 values that is not rotated
// is exact in one), so scores agree with an f32 computation; f32 callers'
// weights do too, f16 callers' are rounded once to f16. That makes 3 (f32: 4)
// MMA passes of the 2 that the operation's flops count, the bound of the
// kernel at 128 channels: 2/3 (1/2) of the tensor cores' rate.
#include "kv8.cuh"
#include "tc.cuh"

namespace sicu {
namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LAZY = 8.0f;
constexpr float LOWEST = -3.402823466e38f;
constexpr float VR_MIN = 9.094947017729282e-13f;      // 2^-40: smaller relative V scales weigh nothing in f16 parts
constexpr uint32_t ALL = 0xffffffffu;

constexpr int PT_ROWS = 256, PT_M = 128, PT_KEYS = 128, PT_BLOCKS = PT_KEYS / KV8_BLOCK;
constexpr int PT_THREADS = 512;       // softmax 2 x 4 warps, K converters 4, MMA issue 1, V converters 3
constexpr int PT_W_K = 8, PT_W_MMA = 12, PT_W_V = 13, PT_NV = 3;
constexpr int PT_RING = 4;            // tiles whose scales are kept

// barriers
enum { B_K_FULL, B_K_FREE, B_V_FULL, B_V_FREE, B_S0, B_S1, B_P0, B_P1, B_OUT, B_DRAIN, B_SC, B_COUNT = B_SC + PT_RING };

template <int HD>
struct PtLay {
    static constexpr int PANELS = HD / 64, PANEL = PT_M * 128;        // 128 rows x 64 halves
    static constexpr int TILE = PANELS * PANEL;
    static constexpr int OFF_Q = 0;                                   // [tile][hi, lo]
    static constexpr int OFF_K = OFF_Q + 4 * TILE;
    static constexpr int OFF_V = OFF_K + TILE;
    static constexpr int OFF_SC = OFF_V + TILE;                       // [ring][8] K scale, V factor, V term
    static constexpr int OFF_RS = OFF_SC + PT_RING * PT_BLOCKS * 16;  // per-row score factor
    static constexpr int OFF_BAR = OFF_RS + PT_ROWS * 4;
    static constexpr int OFF_MISC = OFF_BAR + B_COUNT * 8;
    static constexpr int SMEM = OFF_MISC + 256 + 1024;                // base rounded up to 1024
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float soft_cap(float x, float cap, float inv_cap) {
    const float e = ex2(x * inv_cap * (2.0f * LOG2E));
    return cap - 2.0f * cap * __fdividef(1.0f, 1.0f + fminf(e, 1e30f));
}
__device__ __forceinline__ uint32_t code_pair(uint32_t x, uint32_t sel) {
    const uint32_t h = prmt(x, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), __floats2half2_rn(1152.0f, 1152.0f));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// Bounded wait of all roles: gives up when another role did, or after 2 s,
// with the status bit set.
template <bool POLL = false>
__device__ __forceinline__ bool pt_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status) {
    if (mbar_poll(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!(POLL ? mbar_poll(bar, parity) : mbar_try_wait(bar, parity))) {
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > 2000000000ull) {
            *abort_flag = 1;
            atomicOr(status, STATUS_WAIT_TIMEOUT);
            return false;
        }
    }
    return true;
}

// 32 lanes x 32 columns, not waited for; tie32 after the wait keeps uses behind it
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_all() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tie32(uint32_t (&v)[32]) {
    asm volatile(""
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                   "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :: "memory");
}

// Shared-memory descriptor of V as the N side of O += P V: the keys are the
// K dimension, so N (channels) is the contiguous one. 64 channels of 8 keys
// make one 1024-byte swizzle atom; the next 8 keys follow it (stride offset),
// the next 64 channels come a panel later (leading offset).
__device__ __forceinline__ uint64_t v_desc(uint32_t addr, uint32_t panel) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)SMEM_SWZ_128B << 61);
}

// A converter warp's pieces of a 128-key tile: 16 codes per lane, lanes laid
// so that every eight write 128 bytes without bank conflicts.
template <int HD>
struct Piece {
    static constexpr int ROWS = HD == 128 ? 4 : 8;                    // keys per piece
    static constexpr int COUNT = PT_KEYS / ROWS;
    __device__ static int row(int u, int lane) {
        return HD == 128 ? 4 * u + ((lane >> 2) & 1) + 2 * (lane >> 4) : 8 * u + (lane >> 2);
    }
    __device__ static int panel(int lane) { return HD == 128 ? (lane >> 3) & 1 : 0; }
    __device__ static int quad(int lane) { return lane & 3; }
};
template <int HD>
__device__ __forceinline__ uint4 piece_load(const int8_t *codes, int64_t blk, int u, int lane) {
    using P = Piece<HD>;
    if (blk < 0) return make_uint4(0, 0, 0, 0);
    const int r = P::row(u, lane);
    return __ldg(reinterpret_cast<const uint4 *>(codes + (blk * KV8_BLOCK + (r & 15)) * HD + P::panel(lane) * 64 +
                                                 P::quad(lane) * 16));
}
template <int HD>
__device__ __forceinline__ void piece_store(uint32_t tile, const uint4 &w, int u, int lane) {
    using P = Piece<HD>;
    const int r = P::row(u, lane), q = P::quad(lane);
    const uint32_t base = tile + P::panel(lane) * PtLay<HD>::PANEL + (r >> 3) * 1024 + (r & 7) * 128;
    const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u, c = w.z ^ 0x80808080u, d = w.w ^ 0x80808080u;
    sts128(base + (((2 * q) ^ (r & 7)) << 4), code_pair(a, 0x4140), code_pair(a, 0x4342), code_pair(b, 0x4140), code_pair(b, 0x4342));
    sts128(base + (((2 * q + 1) ^ (r & 7)) << 4), code_pair(c, 0x4140), code_pair(c, 0x4342), code_pair(d, 0x4140), code_pair(d, 0x4342));
}

struct PtParams {
    Kv8Dev c;
    Kv8AttnDev a;
    int skip_rows;        // requests of at most this many rows belong to the other kernel
};

template <typename T, int HD>
__global__ void __launch_bounds__(PT_THREADS, 1) kv8_prompt_kernel(const __grid_constant__ PtParams prm) {
    using Lay = PtLay<HD>;
    constexpr bool SPLIT = sizeof(T) == 4;
    extern __shared__ uint8_t pt_raw[];
    const uint32_t raw = smem_addr(pt_raw), sb = (raw + 1023u) & ~1023u;
    uint8_t *sm = pt_raw + (sb - raw);
    const Kv8Dev &c = prm.c;
    const Kv8AttnDev &a = prm.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sm + Lay::OFF_MISC);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + Lay::OFF_MISC + 4);
    int *found = reinterpret_cast<int *>(sm + Lay::OFF_MISC + 8);             // request, tile
    int *wsum = reinterpret_cast<int *>(sm + Lay::OFF_MISC + 16);             // [16]
    float *wmax = reinterpret_cast<float *>(sm + Lay::OFF_MISC + 80);         // [16]
    float *rsv = reinterpret_cast<float *>(sm + Lay::OFF_RS);
    float4 *sc = reinterpret_cast<float4 *>(sm + Lay::OFF_SC);                // (K scale, V factor, V term, -)
    auto bar = [&](int i) { return sb + Lay::OFF_BAR + 8u * (uint32_t)i; };

    // ---- which request and rows: tiles counted request by request
    const int head = blockIdx.x % c.hkv, want = blockIdx.x / c.hkv, group = a.n_head / c.hkv;
    if (tid == 0) found[0] = -1;
    int before = 0;
    for (int i0 = 0; i0 < a.n_seq; i0 += PT_THREADS) {
        int n = 0;
        if (i0 + tid < a.n_seq) {
            const Kv8Seq s = kv8_seq(a, i0 + tid);
            const int rows = s.n_new * group;
            if (rows > prm.skip_rows) n = (rows + PT_ROWS - 1) / PT_ROWS;
        }
        int x = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(ALL, x, d);
            if (lane >= d) x += y;
        }
        __syncthreads();
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        int base = before, all = before;
        for (int w = 0; w < PT_THREADS / 32; ++w) {
            if (w < warp) base += wsum[w];
            all += wsum[w];
        }
        if (want >= base + x - n && want < base + x) {
            found[0] = i0 + tid;
            // a request's last rows, which see the most keys, first
            found[1] = n - 1 - (want - (base + x - n));
        }
        before = all;
        if (want < before) break;
    }
    __syncthreads();
    if (found[0] < 0) return;
    const int seq = found[0], r0 = found[1] * PT_ROWS;
    const Kv8Seq s = kv8_seq(a, seq);
    const int rows = min(PT_ROWS, s.n_new * group - r0), pos0 = s.len - s.n_new;
    const int n_mt = rows > PT_M ? 2 : 1;
    const int lo = kv8_lo(a, s, pos0 + r0 / group), hi = kv8_hi(s, pos0 + (r0 + rows - 1) / group);
    const int b0 = lo >> 4, b1 = lo < hi ? (hi + 15) >> 4 : b0;
    const int nj = (b1 - b0 + PT_BLOCKS - 1) / PT_BLOCKS;
    T *const out = static_cast<T *>(a.out);
    if (nj == 0) {
        // no row sees a key
        for (int i = tid; i < rows * (HD / 4); i += PT_THREADS) {
            const int r = r0 + i / (HD / 4);
            store4(out + (int64_t)(s.t0 + r / group) * a.out_stride + (int64_t)(head * group + r % group) * HD +
                       i % (HD / 4) * 4, 0.0f, 0.0f, 0.0f, 0.0f);
        }
        return;
    }

    // ---- barriers, tensor memory, the span's largest V scale, q
    if (tid == 0) {
        mbar_init(bar(B_K_FULL), 4);
        mbar_init(bar(B_V_FULL), PT_NV);
        mbar_init(bar(B_P0), 4);
        mbar_init(bar(B_P1), 4);
        for (int i : {B_K_FREE, B_V_FREE, B_S0, B_S1, B_OUT, B_DRAIN}) mbar_init(bar(i), 1);
        for (int i = 0; i < PT_RING; ++i) mbar_init(bar(B_SC + i), 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == PT_W_MMA) tmem_alloc(smem_addr(tmem_slot), 512);
    auto block_of = [&](int b) { return kv8_block(c, kv8_page(c, a, seq, b), head, b & (c.page / KV8_BLOCK - 1)); };
    {
        float m = 0.0f;
        for (int b = b0 + tid; b < b1; b += PT_THREADS) m = fmaxf(m, __ldg(c.vs + block_of(b)));
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(ALL, m, d));
        if (lane == 0) wmax[warp] = m;
    }
    const bool mods = a.cap > 0.0f || a.slopes != nullptr;
    const bool q_lo = SPLIT || a.rope.half > 0;
    {
        // OL lanes per row, one eight-channel piece each
        constexpr int OL = HD / 8, RPW = 32 / OL;
        const T *q = static_cast<const T *>(a.q);
        const int o = lane % OL, neox = a.rope.neox;
        for (int r = warp * RPW + lane / OL; r < PT_ROWS; r += PT_THREADS / 32 * RPW) {
            Oct x;
            if (r < rows) {
                const int t = (r0 + r) / group, h = head * group + (r0 + r) % group;
                const T *src = q + (int64_t)(s.t0 + t) * a.q_stride + (int64_t)h * HD;
                load4(src + oct_a(o, neox), x.a);
                load4(src + oct_b(o, HD, neox), x.b);
                if (a.rope.half) {
                    if (pos0 + t < a.rope.rows) rope_oct(x, a.rope, pos0 + t, o);
                    else if (o == 0) atomicOr(a.status, STATUS_BAD_PLAN);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x.a[e] = x.b[e] = 0.0f;
            }
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fmaxf(fabsf(x.a[e]), fabsf(x.b[e])));
#pragma unroll
            for (int d = 1; d < OL; d <<= 1) m = fmaxf(m, __shfl_xor_sync(ALL, m, d));
            // the row's largest magnitude to [1, 2) by a power of two
            const int e2 = min(max((int)((__float_as_uint(m) >> 23) & 255) - 127, -100), 100);
            const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
            if (o == 0)
                rsv[r] = __uint_as_float((uint32_t)(127 + e2) << 23) *
                         (float)((double)a.scale * (mods ? 1.0 : 1.4426950408889634));
            auto put = [&](int d, const float (&v)[4]) {
                const float v0 = v[0] * inv, v1 = v[1] * inv, v2 = v[2] * inv, v3 = v[3] * inv;
                const uint32_t h0 = half2_bits(v0, v1), h1 = half2_bits(v2, v3);
                const int rr = r & (PT_M - 1);
                const uint32_t at = sb + Lay::OFF_Q + (r / PT_M) * 2 * Lay::TILE + (d >> 6) * Lay::PANEL + (rr >> 3) * 1024 +
                                    (rr & 7) * 128 + ((((d & 63) >> 3) ^ (rr & 7)) << 4) + (d & 4) * 2;
                asm volatile("st.shared.v2.b32 [%0], {%1,%2};" :: "r"(at), "r"(h0), "r"(h1) : "memory");
                asm volatile("st.shared.v2.b32 [%0], {%1,%2};" :: "r"(at + Lay::TILE),
                             "r"(half2_bits(v0 - h2f(h0 & 0xffffu), v1 - h2f(h0 >> 16))),
                             "r"(half2_bits(v2 - h2f(h1 & 0xffffu), v3 - h2f(h1 >> 16))) : "memory");
            };
            put(oct_a(o, neox), x.a);
            put(oct_b(o, HD, neox), x.b);
        }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    float vref = wmax[0];
    for (int w = 1; w < PT_THREADS / 32; ++w) vref = fmaxf(vref, wmax[w]);
    const uint32_t TM_S[2] = {tmem, tmem + 128}, TM_O[2] = {tmem + 256, tmem + 256 + HD};

    if (warp < PT_W_K) {
        // ---- weights: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const int t = warp >> 2, wq = warp & 3, r = t * PT_M + wq * 32 + lane;
        const uint32_t lanes = (uint32_t)(32 * wq) << 16;
        if (t < n_mt) {
            const uint32_t ts = TM_S[t] + lanes, to = TM_O[t] + lanes;
            const bool live = r < rows;
            const int p = pos0 + (r0 + min(r, rows - 1)) / group, h = head * group + (r0 + min(r, rows - 1)) % group;
            const int rlo = kv8_lo(a, s, p), rhi = kv8_hi(s, p);
            // keys all of the warp's rows see
            int wlo = live ? rlo : 0, whi = live ? rhi : INT_MAX;
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                wlo = max(wlo, __shfl_xor_sync(ALL, wlo, d));
                whi = min(whi, __shfl_xor_sync(ALL, whi, d));
            }
            const float rs = rsv[r], inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
            const float slope = a.slopes ? __ldg(a.slopes + h) * LOG2E : 0.0f;
            float m = 0.0f, thr = LOWEST, l = 0.0f;
            bool ok = true;
            for (int j = 0; j < nj; ++j) {
                if (!__all_sync(ALL, pt_wait(bar(B_SC + j % PT_RING), (uint32_t)(j / PT_RING) & 1u, abort_flag, a.status) &&
                                         pt_wait<true>(bar(B_S0 + t), (uint32_t)j & 1u, abort_flag, a.status))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t v[4][32];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, v[q]);
                const float4 *sj = sc + (j % PT_RING) * PT_BLOCKS;
                const int k0 = (b0 + j * PT_BLOCKS) * KV8_BLOCK;
                const bool masked = k0 < wlo || k0 + PT_KEYS > whi;
                tmem_wait_all();
#pragma unroll
                for (int q = 0; q < 4; ++q) tie32(v[q]);
                float cb[PT_BLOCKS];
#pragma unroll
                for (int b = 0; b < PT_BLOCKS; ++b) cb[b] = sj[b].x * rs;
                if (masked || mods) {
                    // scores in place, in powers of two
#pragma unroll
                    for (int b = 0; b < PT_BLOCKS; ++b) {
#pragma unroll
                        for (int e = 0; e < KV8_BLOCK; ++e) {
                            uint32_t &u = v[b >> 1][(b & 1) * 16 + e];
                            const int key = k0 + b * KV8_BLOCK + e;
                            float x = __uint_as_float(u) * cb[b];
                            if (mods) {
                                if (a.cap > 0.0f) x = soft_cap(x, a.cap, inv_cap);
                                x = fmaf(x, LOG2E, -slope * fabsf((float)(p - key)));
                            }
                            u = __float_as_uint(key < rlo || key >= rhi ? -INFINITY : x);
                        }
                        cb[b] = 1.0f;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < PT_BLOCKS; ++b) {
                    float bm = __uint_as_float(v[b >> 1][(b & 1) * 16]);
#pragma unroll
                    for (int e = 1; e < KV8_BLOCK; ++e) bm = fmaxf(bm, __uint_as_float(v[b >> 1][(b & 1) * 16 + e]));
                    mx = fmaxf(mx, bm * cb[b]);
                }
                const bool grow = mx > thr;
                if (__any_sync(ALL, grow)) {
                    float f = 1.0f;
                    if (grow) {
                        if (thr != LOWEST) f = ex2(m - mx);
                        m = mx;
                        thr = mx + LAZY;
                        l *= f;
                    }
                    if (j > 0) {
                        // S of this tile is complete, so every product before it is
#pragma unroll 1
                        for (int q = 0; q < HD; q += 16) {
                            uint32_t w[16];
                            tmem_ld16(to + q, w);
                            tmem_wait_ld(w);
#pragma unroll
                            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
                            tmem_st16(to + q, w);
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t ph[16], pl[SPLIT ? 16 : 1];
#pragma unroll
                    for (int hb = 0; hb < 2; ++hb) {
                        const int b = 2 * q + hb;
                        // f16: the V factor rides in the exponent (term = log2 of
                        // the relative scale) and leaves the sum by its inverse;
                        // f32: a product of its own, exact to 2^-24
                        const float2 fb = make_float2(sj[b].y, sj[b].z);
                        const float sub = SPLIT ? m : m - fb.y;
                        float sum = 0.0f;
#pragma unroll
                        for (int e = 0; e < KV8_BLOCK; e += 2) {
                            const float x0 = ex2(fmaf(__uint_as_float(v[q][hb * 16 + e]), cb[b], -sub));
                            const float x1 = ex2(fmaf(__uint_as_float(v[q][hb * 16 + e + 1]), cb[b], -sub));
                            sum += x0;
                            sum += x1;
                            if constexpr (SPLIT) {
                                const float w0 = x0 * fb.x, w1 = x1 * fb.x;
                                const uint32_t hw = half2_bits(w0, w1);
                                ph[hb * 8 + e / 2] = hw;
                                pl[hb * 8 + e / 2] = half2_bits(w0 - h2f(hw & 0xffffu), w1 - h2f(hw >> 16));
                            } else {
                                ph[hb * 8 + e / 2] = half2_bits(x0, x1);
                            }
                        }
                        l += SPLIT ? sum : sum * fb.x;
                    }
                    tmem_st16(ts + 16 * q, ph);
                    if constexpr (SPLIT) tmem_st16(ts + 64 + 16 * q, pl);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_P0 + t));
            }
            if (ok && __all_sync(ALL, pt_wait<true>(bar(B_OUT), 0, abort_flag, a.status))) {
                tc_fence_after();
                const float f = l == 0.0f ? 0.0f : __fdiv_rn(vref, l);
                const int rr = r0 + r;
                T *dst = out + (int64_t)(s.t0 + rr / group) * a.out_stride + (int64_t)(head * group + rr % group) * HD;
#pragma unroll
                for (int q = 0; q < HD; q += 32) {
                    uint32_t w[32];
                    tmem_ld32(to + q, w);
                    tmem_wait_all();
                    tie32(w);
                    if (live) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            store4(dst + q + e, __uint_as_float(w[e]) * f, __uint_as_float(w[e + 1]) * f,
                                   __uint_as_float(w[e + 2]) * f, __uint_as_float(w[e + 3]) * f);
                    }
                }
            }
        }
    } else {
      // one instruction for each whole warpgroup: 256 x 176 + 256 x 80
      // registers are the launch's 512 x 128
      asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
      if (warp < PT_W_MMA) {
        // ---- K: codes to f16, and the tile's scales
        constexpr int N = Piece<HD>::COUNT / 4;
        const int w = warp - PT_W_K;
        uint4 piece[N];
        int64_t blk = -1;
        float ksc = 0.0f, vsc = 0.0f;
        auto fetch = [&](int j) {
            const int b = b0 + j * PT_BLOCKS + lane;
            blk = -1;
            ksc = vsc = 0.0f;
            if (lane < PT_BLOCKS && b < b1) {
                blk = block_of(b);
                if (w == 0) {
                    ksc = __ldg(c.ks + blk);
                    vsc = __ldg(c.vs + blk);
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int u = w + 4 * i;
                piece[i] = piece_load<HD>(c.k, __shfl_sync(ALL, blk, u * Piece<HD>::ROWS / KV8_BLOCK), u, lane);
            }
        };
        fetch(0);
        for (int j = 0; j < nj; ++j) {
            if (!__all_sync(ALL, pt_wait(bar(B_K_FREE), (uint32_t)(j & 1) ^ 1u, abort_flag, a.status))) break;
#pragma unroll
            for (int i = 0; i < N; ++i) piece_store<HD>(sb + Lay::OFF_K, piece[i], w + 4 * i, lane);
            if (w == 0 && lane < PT_BLOCKS) {
                const float vr = vref > 0.0f ? fmaxf(__fdiv_rn(vsc, vref), VR_MIN) : 1.0f;
                sc[(j % PT_RING) * PT_BLOCKS + lane] =
                    SPLIT ? make_float4(ksc, vr, 0.0f, 0.0f) : make_float4(ksc, __fdiv_rn(1.0f, vr), __log2f(vr), 0.0f);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(B_K_FULL));
                if (w == 0) mbar_arrive(bar(B_SC + j % PT_RING));
            }
            if (j + 1 < nj) fetch(j + 1);
        }
      } else if (warp == PT_W_MMA) {
        // ---- MMA issue
        if (lane == 0) {
            constexpr uint32_t id_s = idesc_f16_f32(PT_M, PT_KEYS), id_o = idesc_f16_f32(PT_M, HD) | (1u << 16);
            auto scores = [&](int t) {
                const uint32_t q = sb + Lay::OFF_Q + t * 2 * Lay::TILE, k = sb + Lay::OFF_K;
                for (int part = 0; part < (q_lo ? 2 : 1); ++part)
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint32_t off = (kk / 4) * Lay::PANEL + (kk % 4) * 32;
                        tc_mma_f16(TM_S[t], smem_desc(q + part * Lay::TILE + off, 1024, SMEM_SWZ_128B),
                                   smem_desc(k + off, 1024, SMEM_SWZ_128B), id_s, (part | kk) != 0);
                    }
                tc_commit(bar(B_S0 + t));
            };
            bool ok = pt_wait<true>(bar(B_K_FULL), 0, abort_flag, a.status);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < n_mt; ++t) scores(t);
                tc_commit(bar(B_K_FREE));
            }
            for (int j = 0; ok && j < nj; ++j) {
                for (int t = 0; ok && t < n_mt; ++t) {
                    if (t == 0) ok = pt_wait<true>(bar(B_V_FULL), (uint32_t)j & 1u, abort_flag, a.status);
                    ok = ok && pt_wait<true>(bar(B_P0 + t), (uint32_t)j & 1u, abort_flag, a.status);
                    if (!ok) break;
                    tc_fence_after();
                    for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
                        for (int kk = 0; kk < PT_KEYS / 16; ++kk)
                            tc_mma_f16_ts(TM_O[t], TM_S[t] + 64 * part + 8 * kk,
                                          v_desc(sb + Lay::OFF_V + kk * 2048, Lay::PANEL), id_o, (j | part | kk) != 0);
                    if (t == n_mt - 1) tc_commit(j + 1 < nj ? bar(B_V_FREE) : bar(B_OUT));
                    if (j + 1 < nj) {
                        if (t == 0) ok = pt_wait<true>(bar(B_K_FULL), (uint32_t)(j + 1) & 1u, abort_flag, a.status);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t);
                        if (t == n_mt - 1) tc_commit(bar(B_K_FREE));
                    }
                }
            }
            if (*abort_flag) {
                // every product issued must end before shared and tensor memory go
                tc_commit(bar(B_DRAIN));
                (void)mbar_wait(bar(B_DRAIN), 0, 200000000ull);
            }
        }
      } else {
        // ---- V: codes to f16
        constexpr int N = (Piece<HD>::COUNT + PT_NV - 1) / PT_NV;
        const int w = warp - PT_W_V;
        uint4 piece[N];
        auto fetch = [&](int j) {
            const int b = b0 + j * PT_BLOCKS + lane;
            int64_t blk = -1;
            if (lane < PT_BLOCKS && b < b1) blk = block_of(b);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int u = w + PT_NV * i;
                const int64_t mine = __shfl_sync(ALL, blk, min(u, Piece<HD>::COUNT - 1) * Piece<HD>::ROWS / KV8_BLOCK);
                if (u < Piece<HD>::COUNT) piece[i] = piece_load<HD>(c.v, mine, u, lane);
            }
        };
        fetch(0);
        for (int j = 0; j < nj; ++j) {
            if (!__all_sync(ALL, pt_wait(bar(B_V_FREE), (uint32_t)(j & 1) ^ 1u, abort_flag, a.status))) break;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (w + PT_NV * i < Piece<HD>::COUNT) piece_store<HD>(sb + Lay::OFF_V, piece[i], w + PT_NV * i, lane);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_V_FULL));
            if (j + 1 < nj) fetch(j + 1);
        }
      }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == PT_W_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int HD>
int launch_typed(const PtParams &p, unsigned ctas, cudaStream_t st) {
    constexpr int smem = PtLay<HD>::SMEM;
    if (cudaFuncSetAttribute(kv8_prompt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return -2;
    kv8_prompt_kernel<T, HD><<<ctas, PT_THREADS, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace

bool kv8_prompt_supported(int hd) { return hd == 64 || hd == 128; }

int launch_kv8_prompt(const Kv8Dev &c, const Kv8AttnDev &a, bool f16, int skip_rows, cudaStream_t st) {
    PtParams p{c, a, skip_rows};
    // at most one partly filled tile per request
    const int64_t rows = (int64_t)a.n_tok * (a.n_head / c.hkv);
    const int64_t ctas = (rows / PT_ROWS + a.n_seq) * c.hkv;
    if (ctas > INT32_MAX) return -1;
    switch (c.hd) {
        case 64: return f16 ? launch_typed<__half, 64>(p, (unsigned)ctas, st) : launch_typed<float, 64>(p, (unsigned)ctas, st);
        case 128: return f16 ? launch_typed<__half, 128>(p, (unsigned)ctas, st) : launch_typed<float, 128>(p, (unsigned)ctas, st);
        default: return -3;
    }
}

}  // namespace sicu
