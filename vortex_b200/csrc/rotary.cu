// Rotary positions, optionally behind an RMS norm of each head, of the queries and keys of an attention layer; the same with
// the keys and values stored in the pages of a cache; and the backward pass.
//
//   xh = x / r, r = sqrt(mean_d x^2 + eps);  u = w * xh  (u = x without a weight);
//   pair i of the first `rot` dimensions turns by t_i = position * inv_freq[i]:
//     y_a = s (u_a cos t_i - u_b sin t_i),  y_b = s (u_a sin t_i + u_b cos t_i);  the other dimensions keep u.
//   backward, with g = the transposed rotation of dy:  dx = (w g - xh mean(w g xh)) / r,  dw = sum over rows of g xh.
//
// Every value is read once and written once, in fp32 between the two, rounded once: memory bounds it, and below some 10^4
// rows the launch.  The vector kernels form the sine and cosine of a (token, pair) once for the heads of a warp, in shared
// memory: up to four steps of 32 / lanes heads side by side (32 16-bit heads of up to 64 values, 16 of 128, 8 of 256, 4 of 512;
// half as many in fp32).  The angle is formed in 64 bits, as turns with the whole turns taken off, since position * inv_freq in
// 32 bits is off by 0.03 rad at position 2^20; what is left, half a turn at most, goes to sincospif as a float.
//
// Measured (bf16, heads of 128, of the measured copy bandwidth; replayed from a graph): 32768 tokens x 64 heads turned in 167 us
// (0.98; 181 as a program's calls on changing inputs, 0.90); 16384 tokens x 40 heads normed and turned in 68 us (0.75: the
// norm's two waits for other lanes, and warps of 8 key heads that are short beside their set-up), backward 100 us (0.77:
// registers, two blocks an SM), in fp32 114 and 173 us (0.90, 0.89); 9757 ragged tokens x 48 heads stored in pages in 50 us
// (0.73); 64 tokens x 64 heads in 2.8 us, stored 3.7 us (the chain position -> table -> store behind the launch).  The general
// kernels form every angle for every head and read value by value: bf16 heads of 80 with 40 turned, 16384 tokens x 40 heads,
// 252 us, normed 346, backward 657 (0.13, 0.09, 0.07); fp32 heads of 512, x 10, 194, 227 and 561 us (0.53, 0.45, 0.27).
#include "attn.cuh"
#include "tma.cuh"
#include "umma.cuh"

VTX_DEFINE_STATUS_READER()

namespace vtx {
namespace {

struct Rows {                    // one of q, k, v: [B, L, H, D] by element strides, unit stride over D
    const void* src;
    int64_t sb, sl, sh;
    void* dst;                   // [B, L, H, D], or pages (see RotArgs::table) [page, slot, H, D]
    int64_t db, dl, dh;
    const void* w;               // norm weight [D] or NULL
    int wd;
    int H;
};

struct RotArgs {
    Rows r[3];                   // q, k, v (v: copied)
    const void* pos;
    int64_t psb, psl;
    const void* freq;
    int pos64, freq64, rot, inter;
    float scale, eps, inv_D;
    int conj;
    int64_t B, L;
    int D;
    // cache: k and v of a token go to page table[seq][position / page_size], slot position % page_size
    int paged;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_ids;
    int64_t table_width, num_seqs, num_pages, page_size;
    // backward
    const void* dy[2];
    int64_t dyb[2], dyl[2], dyh[2];
    float* dw_part;              // rows of D: the queries' blocks, then the keys'
};

constexpr int kThreads = 256;
constexpr int kMaxD = 512;
constexpr int kFwdBlocks = 5, kBwdPerSM = 2, kTokenCost = 1;
constexpr int kBwdBlocks = kNumSMs * 4;

__device__ __forceinline__ int64_t load_pos(const RotArgs& a, int64_t b, int64_t l) {
    const int64_t i = b * a.psb + l * a.psl;
    return a.pos64 ? static_cast<const int64_t*>(a.pos)[i] : (int64_t) static_cast<const int32_t*>(a.pos)[i];
}

// (cos, sin) of position * inv_freq[i], times the scale; the sine negated for the transposed rotation
__device__ __forceinline__ float2 turn(const RotArgs& a, int64_t pos, int i) {
    const double f = a.freq64 ? static_cast<const double*>(a.freq)[i] : (double)static_cast<const float*>(a.freq)[i];
    double t = (double)pos * f * 0.15915494309189533577;      // 1 / (2 pi)
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    return make_float2(c * a.scale, (a.conj ? -s : s) * a.scale);
}

// Where a token's row lies in the pools: its page is loaded when this is made, and looked at when the offset is asked for, so
// that the load can be waited for behind other work.  offset(): elements from the k (which = 1) or v (2) pool's start, or -1
// where the token is not stored: a negative position is padding; one behind its table row, or a page outside the pool, sets the
// status word.
struct Slot {
    int64_t page, slot;
    bool padding;
    __device__ Slot(const RotArgs& a, int64_t tok, int64_t pos) {
        padding = pos < 0;
        page = -1;
        slot = 0;
        if (padding) return;
        const int64_t seq = a.seq_ids ? (int64_t)a.seq_ids[tok] : tok;
        int64_t at;
        if (pos >> 32 | a.page_size >> 32) {
            at = pos / a.page_size;
        } else {                                 // (in 32 bits a tenth of the instructions in front of the load)
            at = (uint32_t)pos / (uint32_t)a.page_size;
        }
        slot = pos - at * a.page_size;
        if (seq >= 0 && seq < a.num_seqs && at < a.table_width) page = a.table[seq * a.table_stride + at];
    }
    __device__ int64_t offset(const RotArgs& a, int which) const {
        if (padding) return -1;
        if (page < 0 || page >= a.num_pages) {
            atomicCAS(&g_device_status, 0, kStatusBadPage);
            return -1;
        }
        return page * a.r[which].db + slot * a.r[which].dl;
    }
};

using umma::f32x2;
using umma::add2;
using umma::fma2;
using umma::mul2;
using umma::pk2;
using umma::sub2;
using umma::up2;

template <typename T> __device__ __forceinline__ float low(uint32_t w);
template <typename T> __device__ __forceinline__ float high(uint32_t w);
template <> __device__ __forceinline__ float low<__nv_bfloat16>(uint32_t w) { return umma::bf_lo(w); }
template <> __device__ __forceinline__ float high<__nv_bfloat16>(uint32_t w) { return umma::bf_hi(w); }
template <> __device__ __forceinline__ float low<__half>(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
template <> __device__ __forceinline__ float high<__half>(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return umma::pack_bf16(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int LANES> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float sum2(f32x2 v) {
    float a, b;
    up2(v, a, b);
    return a + b;
}

// What a lane of the vector kernels holds of a head: N pairs (a[i], b[i]), two values to a 64-bit register and instruction
// (the arithmetic, not the traffic, took the time before: 590 instructions a step of the backward pass).  They come from two
// 16-byte vectors: a from the one and b from the other in the half layout, the even and the odd values of both in the
// interleaved one, which makes all that follows the same for both.
template <typename T, bool INTER> struct Lane {
    static constexpr int N = 16 / sizeof(T), P = N / 2;
    int ea, eb;          // first elements of the two vectors
    bool on, turned;     // inside the head; inside its rotated part
    __device__ int apart() const { return INTER ? N : eb - ea; }
    __device__ Lane(const RotArgs& a, int sub) {
        on = sub * 2 * N < a.D;
        turned = sub * 2 * N < a.rot;
        if (!on) {                                   // (reads what the first lane reads, and writes nothing)
            ea = 0; eb = INTER ? N : 0;
        } else if (INTER) {
            ea = sub * 2 * N; eb = ea + N;
        } else if (turned) {
            ea = sub * N; eb = ea + a.rot / 2;
        } else {                                     // the kept part is halved like the turned one
            ea = a.rot + (sub * 2 * N - a.rot) / 2; eb = ea + (a.D - a.rot) / 2;
        }
    }
    // element of the head that value i of the 2N holds (a first, then b)
    __device__ int element(int i) const { return INTER ? ea + 2 * (i < N ? i : i - N) + (i >= N) : i < N ? ea + i : eb + i - N; }
    __device__ static void unpack(const uint4& u, const uint4& v, f32x2* a, f32x2* b) {
        const uint32_t x[4] = {u.x, u.y, u.z, u.w}, y[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) {
            auto f = [](uint32_t w) { return __uint_as_float(w); };
            if (INTER) {
                a[0] = pk2(f(x[0]), f(x[2])); b[0] = pk2(f(x[1]), f(x[3]));
                a[1] = pk2(f(y[0]), f(y[2])); b[1] = pk2(f(y[1]), f(y[3]));
            } else {
                a[0] = pk2(f(x[0]), f(x[1])); a[1] = pk2(f(x[2]), f(x[3]));
                b[0] = pk2(f(y[0]), f(y[1])); b[1] = pk2(f(y[2]), f(y[3]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (INTER) {
                    const uint32_t p = i < 2 ? x[2 * i] : y[2 * i - 4], q = i < 2 ? x[2 * i + 1] : y[2 * i - 3];
                    a[i] = pk2(low<T>(p), low<T>(q)); b[i] = pk2(high<T>(p), high<T>(q));
                } else {
                    a[i] = pk2(low<T>(x[i]), high<T>(x[i])); b[i] = pk2(low<T>(y[i]), high<T>(y[i]));
                }
            }
        }
    }
    __device__ static void pack(const f32x2* a, const f32x2* b, uint4& u, uint4& v) {
        uint32_t x[4], y[4];
        float a0, a1, b0, b1;
        if constexpr (sizeof(T) == 4) {
            auto w = [](float f) { return __float_as_uint(f); };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                up2(a[i], a0, a1);
                up2(b[i], b0, b1);
                uint32_t* z = i ? y : x;
                if (INTER) { z[0] = w(a0); z[1] = w(b0); z[2] = w(a1); z[3] = w(b1); }
                else { x[2 * i] = w(a0); x[2 * i + 1] = w(a1); y[2 * i] = w(b0); y[2 * i + 1] = w(b1); }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                up2(a[i], a0, a1);
                up2(b[i], b0, b1);
                if (INTER) {
                    uint32_t* z = i < 2 ? x + 2 * i : y + 2 * i - 4;
                    z[0] = pack2<T>(a0, b0); z[1] = pack2<T>(a1, b1);
                } else {
                    x[i] = pack2<T>(a0, a1); y[i] = pack2<T>(b0, b1);
                }
            }
        }
        u = make_uint4(x[0], x[1], x[2], x[3]);
        v = make_uint4(y[0], y[1], y[2], y[3]);
    }
    __device__ static float squares(const f32x2* a, const f32x2* b) {
        f32x2 x = mul2(a[0], a[0]), y = mul2(b[0], b[0]);
#pragma unroll
        for (int i = 1; i < P; ++i) { x = fma2(a[i], a[i], x); y = fma2(b[i], b[i], y); }
        return sum2(add2(x, y));
    }
};

// Values of a head as its lanes hold them, in shared memory: quad q of a lane's at [q][lane], so that the lanes read
// neighbouring 16 bytes.  Not in registers: what hides the memory is the number of warps (five blocks an SM with one step
// loaded ahead 167 us for 32768 tokens x 64 heads; cosines and sines in registers, three blocks and two steps 199).
template <int LANES> __device__ __forceinline__ void load_quad(const float* w, int q, int sub, f32x2& w0, f32x2& w1) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(w + (q * LANES + sub) * 4);
    w0 = v.x;
    w1 = v.y;
}
// The weights: 2N values a lane.
template <typename T, bool INTER, int LANES> __device__ __forceinline__ void stage_weights(const RotArgs& a, const Rows& r, float* dst) {
    if (!r.w) return;
    for (int i = threadIdx.x; i < Lane<T, INTER>::N * 2 * LANES; i += kThreads) {
        const int q = i / (4 * LANES), sub = i / 4 % LANES;
        const Lane<T, INTER> ln(a, sub);
        dst[i] = ln.on ? ld_param(r.w, r.wd, ln.element(q * 4 + i % 4)) : 0.f;
    }
}
// Cosines, then sines, of a token's pairs, N values a lane each, in the warp's own piece.
template <int N, int LANES> __device__ __forceinline__ void stage_turns(const RotArgs& a, float* dst, int64_t pos) {
    __syncwarp();
    for (int i = threadIdx.x & 31; i < a.rot / 2; i += 32) {
        const float2 cs = turn(a, pos, i);
        float* d = dst + (i % N / 4 * LANES + i / N) * 4 + i % 4;
        d[0] = cs.x;
        d[N * LANES] = cs.y;
    }
    __syncwarp();
}
template <int N, int LANES> __device__ __forceinline__ void rotate(const float* turns, int sub, f32x2* a, f32x2* b) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        f32x2 c[2], s[2];
        load_quad<LANES>(turns, q, sub, c[0], c[1]);
        load_quad<LANES>(turns + N * LANES, q, sub, s[0], s[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const f32x2 x = a[2 * q + j], y = b[2 * q + j];
            a[2 * q + j] = sub2(mul2(x, c[j]), mul2(y, s[j]));
            b[2 * q + j] = fma2(x, s[j], mul2(y, c[j]));
        }
    }
}

// A warp takes one token and `chunk` heads of its queries, keys or values, 32 / LANES heads side by side (LANES lanes cover a
// head).  No warp waits for another (but for the weights, once): a token's chain position -> angles, page lookup -> store
// hides behind the other warps' traffic.
struct Chunks { int size, q, k, v; };      // heads in one; chunks of a token's queries, keys, values

template <typename T, bool INTER, int LANES>
__global__ void __launch_bounds__(kThreads, kFwdBlocks) rotary_fwd_kernel(const __grid_constant__ RotArgs a, const __grid_constant__ Chunks ch) {
    using Ln = Lane<T, INTER>;
    constexpr int N = Ln::N, P = Ln::P, STEP = 32 / LANES;
    __shared__ __align__(16) float s_turn[kThreads / 32][2 * N * LANES], s_w[2][2 * N * LANES];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES, slot = lane / LANES;
    const bool any_norm = a.r[0].w || a.r[1].w;
    const uint32_t item = blockIdx.x * (kThreads / 32) + warp, per = ch.q + ch.k + ch.v, tok = item / per, L = (uint32_t)a.L;
    const bool live = tok < (uint32_t)(a.B * a.L);
    int c = (int)(item - tok * per);
    const int which = c < ch.q ? 0 : c < ch.q + ch.k ? 1 : 2;
    c -= which == 0 ? 0 : which == 1 ? ch.q : ch.q + ch.k;
    const Rows& r = a.r[which];
    const uint32_t b = live ? tok / L : 0, l = live ? tok - b * L : 0;     // (a warp behind the last token reads the first)
    const int first = c * ch.size, count = ch.size < r.H - first ? ch.size : r.H - first;
    const Ln ln(a, sub);
    const int apart = ln.apart();
    const T* const head0 = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + first * r.sh + ln.ea;
    const T* src = head0 + slot * r.sh;
    const int64_t src_step = STEP * r.sh, dst_step = STEP * r.dh;
    uint4 nu, nv;                                                  // loaded a step ahead
    // (a lane behind the last head reads the first: every address lies inside the rows)
    auto fetch = [&](int h0) {
        const T* p = h0 + STEP > count && h0 + slot >= count ? head0 : src;
        nu = *reinterpret_cast<const uint4*>(p);
        nv = *reinterpret_cast<const uint4*>(p + apart);
        src += src_step;
    };
    fetch(0);
    if (any_norm) {
        stage_weights<T, INTER, LANES>(a, a.r[0], s_w[0]);
        stage_weights<T, INTER, LANES>(a, a.r[1], s_w[1]);
        __syncthreads();
    }
    if (!live) return;
    const int64_t pos = load_pos(a, b, l);
    const bool paged = a.paged && which;
    const Slot where(a, tok, paged ? pos : -1);
    if (which < 2) stage_turns<N, LANES>(a, s_turn[warp], pos);
    const int64_t at = paged ? where.offset(a, which) : b * r.db + l * r.dl;
    if (paged && at < 0) return;
    T* dst = static_cast<T*>(r.dst) + at + (first + slot) * r.dh + ln.ea;
    const bool norm = which < 2 && r.w;
    for (int h0 = 0; h0 < count; h0 += STEP) {
        uint4 u = nu, v = nv;
        if (h0 + STEP < count) fetch(h0 + STEP);
        if (which < 2) {
            f32x2 xa[P], xb[P];
            Ln::unpack(u, v, xa, xb);
            if (norm) {
                const float ss = group_sum<LANES>(ln.on ? Ln::squares(xa, xb) : 0.f);
                const float inv = rsqrtf(ss * a.inv_D + a.eps);
                const f32x2 inv2 = pk2(inv, inv);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    f32x2 w0, w1;
                    load_quad<LANES>(s_w[which], q, sub, w0, w1);
                    f32x2* x = (q < P / 2 ? xa : xb) + 2 * (q % (P / 2));
                    x[0] = mul2(mul2(x[0], inv2), w0);
                    x[1] = mul2(mul2(x[1], inv2), w1);
                }
            }
            if (ln.turned) rotate<N, LANES>(s_turn[warp], sub, xa, xb);
            Ln::pack(xa, xb, u, v);
        }
        if (ln.on && h0 + slot < count) {
            *reinterpret_cast<uint4*>(dst) = u;
            *reinterpret_cast<uint4*>(dst + apart) = v;
        }
        dst += dst_step;
    }
}

// Backward behind a norm.  The first blocks take the queries, the rest the keys; a warp walks its tokens, all heads of one
// before the next.  A lane keeps its dimensions through all rows, so the weight's gradient gathers in its registers, then
// across the block, and leaves as one row of partial sums per block: summed in a fixed order, no atomics.
template <typename T, bool INTER, int LANES>
__global__ void __launch_bounds__(kThreads, kBwdPerSM) rotary_bwd_kernel(const __grid_constant__ RotArgs a, int q_blocks) {
    using Ln = Lane<T, INTER>;
    constexpr int N = Ln::N, P = Ln::P, STEP = 32 / LANES;
    __shared__ __align__(16) float s_turn[kThreads / 32][2 * N * LANES], s_w[2 * N * LANES], s_sum[kThreads / 32][2 * N * LANES];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES, slot = lane / LANES;
    const int which = (int)blockIdx.x >= q_blocks;
    const Rows& r = a.r[which];
    const uint32_t tokens = (uint32_t)(a.B * a.L), L = (uint32_t)a.L;
    const uint32_t warps = (which ? gridDim.x - q_blocks : q_blocks) * (kThreads / 32);
    const bool norm = r.w;
    const Ln ln(a, sub);
    const int apart = ln.apart(), heads = r.H;
    const int64_t x_head = r.sh, g_head = a.dyh[which], d_head = r.dh;
    f32x2 dwa[P], dwb[P];
#pragma unroll
    for (int i = 0; i < P; ++i) dwa[i] = dwb[i] = pk2(0.f, 0.f);
    stage_weights<T, INTER, LANES>(a, r, s_w);
    __syncthreads();
    const T *x0 = nullptr, *g0 = nullptr, *xp = nullptr, *gp = nullptr;     // a token's first head, and the lane's next
    uint4 nga, ngb, nva, nvb;                                      // loaded a step ahead, across tokens
    auto begin = [&](uint32_t t) {
        const uint32_t b = t / L, l = t - b * L;
        x0 = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + ln.ea;
        g0 = static_cast<const T*>(a.dy[which]) + b * a.dyb[which] + l * a.dyl[which] + ln.ea;
        xp = x0 + slot * x_head;
        gp = g0 + slot * g_head;
    };
    // (a lane behind the last head reads the first: every address lies inside the rows)
    auto fetch = [&](int h0) {
        const bool in = h0 + STEP <= heads || h0 + slot < heads;
        const T* g = in ? gp : g0;
        nga = *reinterpret_cast<const uint4*>(g);
        ngb = *reinterpret_cast<const uint4*>(g + apart);
        gp += STEP * g_head;
        if (norm) {
            const T* x = in ? xp : x0;
            nva = *reinterpret_cast<const uint4*>(x);
            nvb = *reinterpret_cast<const uint4*>(x + apart);
            xp += STEP * x_head;
        }
    };
    const uint32_t t0 = (blockIdx.x - (which ? q_blocks : 0)) * (kThreads / 32) + warp;
    int64_t next_pos = 0;
    if (t0 < tokens) {
        begin(t0);
        fetch(0);
        next_pos = load_pos(a, t0 / L, t0 % L);
    }
    for (uint32_t t = t0; t < tokens; t += warps) {
        const uint32_t b = t / L, l = t - b * L, n = t + warps;
        T* dp = static_cast<T*>(r.dst) + b * r.db + l * r.dl + slot * d_head + ln.ea;
        const int64_t pos = next_pos;
        if (n < tokens) next_pos = load_pos(a, n / L, n % L);
        stage_turns<N, LANES>(a, s_turn[warp], pos);
        for (int h0 = 0; h0 < heads; h0 += STEP) {
            const bool mine = ln.on && h0 + slot < heads;
            uint4 ga = nga, gb = ngb;
            const uint4 va = nva, vb = nvb;
            if (h0 + STEP < heads) {
                fetch(h0 + STEP);
            } else if (n < tokens) {
                begin(n);
                fetch(0);
            }
            f32x2 da[P], db[P];
            if (norm) {
                f32x2 xa[P], xb[P];
                Ln::unpack(va, vb, xa, xb);
                const float ss = group_sum<LANES>(ln.on ? Ln::squares(xa, xb) : 0.f);
                const float inv = rsqrtf(ss * a.inv_D + a.eps);
                const f32x2 inv2 = pk2(inv, inv);
                Ln::unpack(ga, gb, da, db);
                if (ln.turned) rotate<N, LANES>(s_turn[warp], sub, da, db);
                f32x2 dot2 = pk2(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    f32x2 wq[2];
                    load_quad<LANES>(s_w, q, sub, wq[0], wq[1]);
                    const int at = 2 * (q % (P / 2));
                    f32x2 *x2 = (q < P / 2 ? xa : xb) + at, *d = (q < P / 2 ? da : db) + at, *dw = (q < P / 2 ? dwa : dwb) + at;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        x2[j] = mul2(x2[j], inv2);                          // xh
                        if (mine) dw[j] = fma2(d[j], x2[j], dw[j]);
                        d[j] = mul2(d[j], wq[j]);                           // w g
                        dot2 = fma2(d[j], x2[j], dot2);
                    }
                }
                const float mean = group_sum<LANES>(ln.on ? sum2(dot2) : 0.f) * -a.inv_D;
                const f32x2 mean2 = pk2(mean, mean);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    da[j] = mul2(fma2(mean2, xa[j], da[j]), inv2);
                    db[j] = mul2(fma2(mean2, xb[j], db[j]), inv2);
                }
            } else {
                Ln::unpack(ga, gb, da, db);
                if (ln.turned) rotate<N, LANES>(s_turn[warp], sub, da, db);
            }
            if (mine) {
                Ln::pack(da, db, ga, gb);
                *reinterpret_cast<uint4*>(dp) = ga;
                *reinterpret_cast<uint4*>(dp + apart) = gb;
            }
            dp += STEP * d_head;
        }
    }
    // the sums of a lane's values: over the warp's rows, then the warps
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float x[4];
        up2(dwa[j / 2], x[0], x[1]);
        up2(dwb[j / 2], x[2], x[3]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float v = x[2 * k + j % 2];
#pragma unroll
            for (int o = LANES; o < 32; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (slot == 0) s_sum[warp][sub * 2 * N + k * N + j] = v;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * N * LANES; i += kThreads) {
        const Ln own(a, i / (2 * N));
        float sum = 0.f;
        for (int w = 0; w < kThreads / 32; ++w) sum += s_sum[w][i];
        if (own.on) a.dw_part[(int64_t)blockIdx.x * a.D + own.element(i % (2 * N))] = sum;
    }
}

// Any head size and alignment (heads or rotated parts that are no whole pairs of 16-byte vectors, as 40 of 80 16-bit values, or
// that have more than 32 of them; rows off 16-byte boundaries): a warp per (token, head), values one by one.  Pair i, and the kept dimensions behind the
// pairs, belong to lane i % 32 in both passes, which is what lets a row be rewritten in place.
struct Pairs {
    int half, rot, D, inter;
    __device__ int count() const { return half + (D - rot); }
    __device__ bool get(int i, int& p, int& q) const {               // false: one kept dimension, p
        if (i >= half) { p = rot + (i - half); q = p; return false; }
        p = inter ? 2 * i : i; q = inter ? 2 * i + 1 : i + half;
        return true;
    }
};

template <typename T> __global__ void __launch_bounds__(kThreads) rotary_fwd_any_kernel(const __grid_constant__ RotArgs a) {
    const int lane = threadIdx.x & 31;
    const int heads = a.r[0].H + a.r[1].H + a.r[2].H;
    const int64_t id = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (id >= a.B * a.L * heads) return;
    const int64_t tok = id / heads, b = tok / a.L, l = tok - b * a.L;
    int h = (int)(id - tok * heads);
    const int which = h < a.r[0].H ? 0 : h < a.r[0].H + a.r[1].H ? 1 : 2;
    h -= which == 0 ? 0 : which == 1 ? a.r[0].H : a.r[0].H + a.r[1].H;
    const Rows& r = a.r[which];
    const T* x = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + h * r.sh;
    const int64_t pos = load_pos(a, b, l);
    T* y = static_cast<T*>(r.dst) + h * r.dh;
    if (a.paged && which) {
        const int64_t at = Slot(a, tok, pos).offset(a, which);
        if (at < 0) return;
        y += at;
    } else {
        y += b * r.db + l * r.dl;
    }
    if (which == 2) {
        for (int d = lane; d < a.D; d += 32) y[d] = x[d];
        return;
    }
    float inv = 1.f;
    if (r.w) {
        float ss = 0.f;
        for (int d = lane; d < a.D; d += 32) ss += to_f32<T>(x[d]) * to_f32<T>(x[d]);
        inv = rsqrtf(group_sum<32>(ss) / (float)a.D + a.eps);
    }
    const Pairs ps{a.rot / 2, a.rot, a.D, a.inter};
    for (int i = lane; i < ps.count(); i += 32) {
        int p, q;
        const bool pair = ps.get(i, p, q);
        float xp = to_f32<T>(x[p]), xq = to_f32<T>(x[q]);
        if (r.w) { xp *= inv * ld_param(r.w, r.wd, p); xq *= inv * ld_param(r.w, r.wd, q); }
        if (pair) {
            const float2 cs = turn(a, pos, i);
            y[p] = from_f32<T>(xp * cs.x - xq * cs.y);
            y[q] = from_f32<T>(xp * cs.y + xq * cs.x);
        } else {
            y[p] = from_f32<T>(xp);
        }
    }
}

template <typename T> __global__ void __launch_bounds__(kThreads) rotary_bwd_any_kernel(const __grid_constant__ RotArgs a) {
    extern __shared__ float s_dw[];                                // [warp][2][D]; a dimension of it belongs to one lane
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kThreads / 32;
    float* mine = s_dw + (int64_t)warp * 2 * a.D;
    for (int i = threadIdx.x; i < warps * 2 * a.D; i += kThreads) s_dw[i] = 0.f;
    __syncthreads();
    const Pairs ps{a.rot / 2, a.rot, a.D, a.inter};
    const int heads = a.r[0].H + a.r[1].H;
    for (int64_t id = (int64_t)blockIdx.x * warps + warp; id < a.B * a.L * heads; id += (int64_t)gridDim.x * warps) {
        const int64_t tok = id / heads, b = tok / a.L, l = tok - b * a.L;
        int h = (int)(id - tok * heads);
        const int which = h >= a.r[0].H;
        h -= which ? a.r[0].H : 0;
        const Rows& r = a.r[which];
        const T* x = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + h * r.sh;
        const T* dy = static_cast<const T*>(a.dy[which]) + b * a.dyb[which] + l * a.dyl[which] + h * a.dyh[which];
        T* dx = static_cast<T*>(r.dst) + b * r.db + l * r.dl + h * r.dh;
        const int64_t pos = load_pos(a, b, l);
        float inv = 1.f, back = 0.f;
        for (int pass = 0; pass < 2; ++pass) {
            float ss = 0.f, dot = 0.f;
            if (pass == 0 && !r.w) continue;
            for (int i = lane; i < ps.count(); i += 32) {
                int p, q;
                const bool pair = ps.get(i, p, q);
                float gp = to_f32<T>(dy[p]), gq = to_f32<T>(dy[q]);
                if (pair) {
                    const float2 cs = turn(a, pos, i);
                    const float t = gp * cs.x - gq * cs.y;
                    gq = gp * cs.y + gq * cs.x;
                    gp = t;
                }
                const float xp = to_f32<T>(x[p]), xq = to_f32<T>(x[q]);
                const float wp = r.w ? ld_param(r.w, r.wd, p) : 1.f, wq = r.w ? ld_param(r.w, r.wd, q) : 1.f;
                if (pass == 0) {
                    ss += xp * xp + (pair ? xq * xq : 0.f);
                    dot += wp * gp * xp + (pair ? wq * gq * xq : 0.f);
                    continue;
                }
                if (r.w) {
                    mine[which * a.D + p] += gp * xp * inv;
                    if (pair) mine[which * a.D + q] += gq * xq * inv;
                    gp = inv * (wp * gp - back * xp);
                    gq = inv * (wq * gq - back * xq);
                }
                dx[p] = from_f32<T>(gp);
                if (pair) dx[q] = from_f32<T>(gq);
            }
            if (pass == 0) {
                inv = rsqrtf(group_sum<32>(ss) / (float)a.D + a.eps);
                back = group_sum<32>(dot) * inv * inv / (float)a.D;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) {
        const int which = i >= a.D;
        float s = 0.f;
        for (int w = 0; w < warps; ++w) s += s_dw[(int64_t)w * 2 * a.D + i];
        a.dw_part[((int64_t)which * gridDim.x + blockIdx.x) * a.D + (i - which * a.D)] = s;
    }
}

// Partial sums, q_rows rows of D for the queries and k_rows for the keys, -> the two weight gradients in the weights' types.
// Block (x, which): 32 values, 32 rows of them at a time.  (A warp per value read 32 lines for 32 numbers: 6.9 us.)
__global__ void __launch_bounds__(1024) rotary_dw_kernel(const float* part, int q_rows, int k_rows, int D, void* dwq, int qd, void* dwk, int kd) {
    __shared__ float s_sum[32][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, at = blockIdx.x * 32 + lane, key = blockIdx.y;
    void* out = key ? dwk : dwq;
    if (!out) return;
    const int rows = key ? k_rows : q_rows, code = key ? kd : qd;
    const float* p = part + (key ? (int64_t)q_rows * D : 0);
    float s = 0.f;
    if (at < D)
#pragma unroll 4
        for (int b = row; b < rows; b += 32) s += p[(int64_t)b * D + at];
    s_sum[row][lane] = s;
    __syncthreads();
    s = group_sum<32>(s_sum[lane][row]);                           // (warp `row` now holds one value's 32 sums)
    const int i = blockIdx.x * 32 + row;
    if (lane || i >= D) return;
    if (code == VTX_F32) static_cast<float*>(out)[i] = s;
    else if (code == VTX_BF16) static_cast<__nv_bfloat16*>(out)[i] = from_f32<__nv_bfloat16>(s);
    else static_cast<__half*>(out)[i] = from_f32<__half>(s);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
bool rows_aligned(const void* p, int64_t sb, int64_t sl, int64_t sh, int64_t es) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (sb * es) % 16 == 0 && (sl * es) % 16 == 0 && (sh * es) % 16 == 0;
}

// Lanes of a head in the vector kernels: 4, 8, 16 or 32; 0 where they do not apply: heads and their rotated part in whole
// pairs of 16-byte vectors, at most 32 pairs to a head, all rows on 16-byte boundaries.
int vector_lanes(const RotArgs& a, int64_t es) {
    const int pair = 2 * (int)(16 / es);
    if (a.D % pair || a.rot % pair || a.D / pair > 32) return 0;
    for (int i = 0; i < 3; ++i) {
        const Rows& r = a.r[i];
        if (r.H && (!rows_aligned(r.src, r.sb, r.sl, r.sh, es) || !rows_aligned(r.dst, r.db, r.dl, r.dh, es))) return 0;
        if (i < 2 && r.H && a.dy[i] && !rows_aligned(a.dy[i], a.dyb[i], a.dyl[i], a.dyh[i], es)) return 0;
    }
    int lanes = 4;
    while (lanes * pair < a.D) lanes *= 2;
    return lanes;
}

#define VTX_DISPATCH_LANES(lanes, N, ...)                        \
    switch (lanes) {                                             \
        case 4:  { constexpr int N = 4;  __VA_ARGS__; break; }   \
        case 8:  { constexpr int N = 8;  __VA_ARGS__; break; }   \
        case 16: { constexpr int N = 16; __VA_ARGS__; break; }   \
        default: { constexpr int N = 32; __VA_ARGS__; break; }   \
    }

int launch_fwd(const RotArgs& a, int64_t io, cudaStream_t s, const char* who) {
    const int64_t tokens = a.B * a.L, heads = a.r[0].H + a.r[1].H + a.r[2].H;
    if (tokens == 0 || heads == 0) return VTX_OK;
    const int lanes = vector_lanes(a, dtype_size(io));
    if (!lanes) {
        const int64_t blocks = ceil_div<int64_t>(tokens * heads, kThreads / 32);
        VTX_REQUIRE(blocks < ((int64_t)1 << 31), VTX_ERR_UNSUPPORTED, "%s: more than 2^34 rows", who);
        VTX_DISPATCH_IO(io, T, rotary_fwd_any_kernel<T><<<(unsigned)blocks, kThreads, 0, s>>>(a));
        return check_launch(who);
    }
    // up to four steps a warp once that still gives every SM its warps; below, fewer, down to one
    const int step = 32 / lanes;
    int steps = 4;
    auto chunks = [&](int h) { return (int)ceil_div<int64_t>(h, steps * step); };
    auto per_token = [&] { return (int64_t)chunks(a.r[0].H) + chunks(a.r[1].H) + chunks(a.r[2].H); };
    while (steps > 1 && tokens * per_token() < (int64_t)kNumSMs * kFwdBlocks * (kThreads / 32)) steps /= 2;
    const Chunks ch{steps * step, chunks(a.r[0].H), chunks(a.r[1].H), chunks(a.r[2].H)};
    const int64_t items = tokens * per_token(), blocks = ceil_div<int64_t>(items, kThreads / 32);
    VTX_REQUIRE(items < ((int64_t)1 << 32) - kThreads, VTX_ERR_UNSUPPORTED, "%s: more than 2^32 pieces of heads", who);
    VTX_DISPATCH_IO(io, T, VTX_DISPATCH_LANES(lanes, N, {
        if (a.inter) rotary_fwd_kernel<T, true, N><<<(unsigned)blocks, kThreads, 0, s>>>(a, ch);
        else rotary_fwd_kernel<T, false, N><<<(unsigned)blocks, kThreads, 0, s>>>(a, ch);
    }));
    return check_launch(who);
}

int fill(RotArgs& a, const vtx_rotary_params& p, const char* who) {
    VTX_REQUIRE(valid_dtype(p.io_dtype), VTX_ERR_BAD_ARG, "%s: unknown io dtype %lld", who, (long long)p.io_dtype);
    VTX_REQUIRE(p.B >= 0 && p.L >= 0 && p.Hq >= 0 && p.Hk >= 0 && p.D > 0, VTX_ERR_BAD_ARG, "%s: negative size", who);
    VTX_REQUIRE(p.D <= kMaxD, VTX_ERR_UNSUPPORTED, "%s: heads of %lld > %d values", who, (long long)p.D, kMaxD);
    VTX_REQUIRE(p.Hq < (1 << 20) && p.Hk < (1 << 20), VTX_ERR_UNSUPPORTED, "%s: more than 2^20 heads", who);
    VTX_REQUIRE(p.rot >= 0 && p.rot % 2 == 0 && p.rot <= p.D, VTX_ERR_BAD_ARG, "%s: %lld rotated of %lld values of a head", who,
                (long long)p.rot, (long long)p.D);
    const bool any = p.B > 0 && p.L > 0;
    VTX_REQUIRE(!any || (p.B < ((int64_t)1 << 31) && p.L < ((int64_t)1 << 31) && p.B * p.L < ((int64_t)1 << 31)), VTX_ERR_UNSUPPORTED,
                "%s: more than 2^31 tokens", who);
    VTX_REQUIRE(!any || !p.Hq || p.q, VTX_ERR_BAD_ARG, "%s: null pointer", who);
    VTX_REQUIRE(!any || !p.Hk || p.k, VTX_ERR_BAD_ARG, "%s: null pointer", who);
    VTX_REQUIRE(!any || (p.positions && (p.inv_freq || !p.rot)), VTX_ERR_BAD_ARG, "%s: null pointer", who);
    VTX_REQUIRE((!p.q_weight || valid_dtype(p.q_weight_dtype)) && (!p.k_weight || valid_dtype(p.k_weight_dtype)), VTX_ERR_BAD_ARG,
                "%s: unknown weight dtype", who);
    a.r[0] = Rows{p.q, p.q_stride_b, p.q_stride_l, p.q_stride_h, p.q_out, p.q_out_stride_b, p.q_out_stride_l, p.q_out_stride_h,
                  p.q_weight, (int)p.q_weight_dtype, (int)p.Hq};
    a.r[1] = Rows{p.k, p.k_stride_b, p.k_stride_l, p.k_stride_h, p.k_out, p.k_out_stride_b, p.k_out_stride_l, p.k_out_stride_h,
                  p.k_weight, (int)p.k_weight_dtype, (int)p.Hk};
    a.pos = p.positions; a.pos64 = p.positions_i64 != 0; a.psb = p.pos_stride_b; a.psl = p.pos_stride_l;
    a.freq = p.inv_freq; a.freq64 = p.inv_freq_f64 != 0; a.rot = (int)p.rot; a.inter = p.interleaved != 0;
    a.scale = (float)p.scale; a.eps = (float)p.eps; a.conj = 0;
    a.B = p.B; a.L = p.L; a.D = (int)p.D; a.inv_D = 1.f / (float)p.D;
    return VTX_OK;
}

}  // namespace
}  // namespace vtx

extern "C" int vtx_qk_norm_rotary_fwd(const vtx_rotary_params* p, void* stream) {
    using namespace vtx;
    VTX_REQUIRE(p, VTX_ERR_BAD_ARG, "qk_norm_rotary: null pointer");
    RotArgs a{};
    if (int rc = fill(a, *p, "qk_norm_rotary")) return rc;
    const bool any = p->B > 0 && p->L > 0;
    VTX_REQUIRE(!any || ((!p->Hq || p->q_out) && (!p->Hk || p->k_out)), VTX_ERR_BAD_ARG, "qk_norm_rotary: null pointer");
    return launch_fwd(a, p->io_dtype, (cudaStream_t)stream, "qk_norm_rotary");
}

extern "C" int64_t vtx_qk_norm_rotary_bwd_scratch_bytes(const vtx_rotary_params* p) {
    return p && (p->q_weight || p->k_weight) && p->D > 0 ? (int64_t)vtx::kBwdBlocks * 2 * p->D * 4 : 0;
}

extern "C" int vtx_qk_norm_rotary_bwd(const vtx_rotary_bwd_params* p, void* stream) {
    using namespace vtx;
    VTX_REQUIRE(p, VTX_ERR_BAD_ARG, "qk_norm_rotary_bwd: null pointer");
    const vtx_rotary_params& f = p->fwd;
    RotArgs a{};
    if (int rc = fill(a, f, "qk_norm_rotary_bwd")) return rc;
    const int64_t tokens = f.B * f.L;
    const bool norm = f.q_weight || f.k_weight;
    VTX_REQUIRE(!tokens || ((!f.Hq || (p->dq_out && f.q_out)) && (!f.Hk || (p->dk_out && f.k_out))), VTX_ERR_BAD_ARG,
                "qk_norm_rotary_bwd: null pointer");
    a.conj = 1;
    cudaStream_t s = (cudaStream_t)stream;
    if (!norm) {                                     // the transposed rotation of dy: the forward kernel on other rows
        a.r[0].src = p->dq_out; a.r[0].sb = p->dq_out_stride_b; a.r[0].sl = p->dq_out_stride_l; a.r[0].sh = p->dq_out_stride_h;
        a.r[1].src = p->dk_out; a.r[1].sb = p->dk_out_stride_b; a.r[1].sl = p->dk_out_stride_l; a.r[1].sh = p->dk_out_stride_h;
        return launch_fwd(a, f.io_dtype, s, "qk_norm_rotary_bwd");
    }
    VTX_REQUIRE(p->scratch, VTX_ERR_BAD_ARG, "qk_norm_rotary_bwd: scratch needed (vtx_qk_norm_rotary_bwd_scratch_bytes)");
    VTX_REQUIRE((!f.q_weight || p->dq_weight) && (!f.k_weight || p->dk_weight), VTX_ERR_BAD_ARG, "qk_norm_rotary_bwd: null weight gradient");
    a.dy[0] = p->dq_out; a.dyb[0] = p->dq_out_stride_b; a.dyl[0] = p->dq_out_stride_l; a.dyh[0] = p->dq_out_stride_h;
    a.dy[1] = p->dk_out; a.dyb[1] = p->dk_out_stride_b; a.dyl[1] = p->dk_out_stride_l; a.dyh[1] = p->dk_out_stride_h;
    a.dw_part = static_cast<float*>(p->scratch);
    int64_t q_rows = 0, k_rows = 0;
    if (tokens && f.Hq + f.Hk) {
        const int lanes = vector_lanes(a, dtype_size(f.io_dtype));
        if (!lanes) {
            const int64_t warps = ceil_div<int64_t>(tokens * (f.Hq + f.Hk), kThreads / 32);
            q_rows = k_rows = warps < kBwdBlocks ? warps : kBwdBlocks;
            VTX_DISPATCH_IO(f.io_dtype, T,
                            rotary_bwd_any_kernel<T><<<(unsigned)q_rows, kThreads, (size_t)(kThreads / 32) * 2 * f.D * 4, s>>>(a));
        } else {
            // blocks for queries and keys in proportion to their heads, a warp at least a token
            const int64_t most = ceil_div<int64_t>(tokens, kThreads / 32), total = kNumSMs * kBwdPerSM;
            auto cost = [&](int64_t h) { return h ? ceil_div<int64_t>(h, 32 / lanes) + kTokenCost : 0; };
            q_rows = f.Hq ? (total * cost(f.Hq) + (cost(f.Hq) + cost(f.Hk)) / 2) / (cost(f.Hq) + cost(f.Hk)) : 0;
            if (f.Hq) q_rows = q_rows < 1 ? 1 : f.Hk && q_rows > total - 1 ? total - 1 : q_rows;
            k_rows = f.Hk ? total - q_rows : 0;
            q_rows = q_rows < most ? q_rows : most;
            k_rows = k_rows < most ? k_rows : most;
            const unsigned blocks = (unsigned)(q_rows + k_rows);
            VTX_DISPATCH_IO(f.io_dtype, T, VTX_DISPATCH_LANES(lanes, N, {
                if (a.inter) rotary_bwd_kernel<T, true, N><<<blocks, kThreads, 0, s>>>(a, (int)q_rows);
                else rotary_bwd_kernel<T, false, N><<<blocks, kThreads, 0, s>>>(a, (int)q_rows);
            }));
        }
    }
    if (q_rows + k_rows)
        if (int rc = check_launch("qk_norm_rotary_bwd")) return rc;
    rotary_dw_kernel<<<dim3((unsigned)ceil_div<int64_t>(f.D, 32), 2), 1024, 0, s>>>(
        a.dw_part, (int)q_rows, (int)k_rows, (int)f.D, f.q_weight ? p->dq_weight : nullptr, (int)f.q_weight_dtype,
        f.k_weight ? p->dk_weight : nullptr, (int)f.k_weight_dtype);
    return check_launch("qk_norm_rotary_bwd");
}

extern "C" int vtx_rotary_append(const vtx_rotary_append_params* p, void* stream) {
    using namespace vtx;
    VTX_REQUIRE(p, VTX_ERR_BAD_ARG, "rotary_append: null pointer");
    RotArgs a{};
    const vtx_rotary_params& f = p->rot;
    if (int rc = fill(a, f, "rotary_append")) return rc;
    const int64_t tokens = f.B * f.L;
    VTX_REQUIRE(f.Hk > 0, VTX_ERR_BAD_ARG, "rotary_append: no key heads");
    VTX_REQUIRE(p->page_size > 0 && p->num_pages >= 0 && p->num_seqs >= 0 && p->table_width >= 0, VTX_ERR_BAD_ARG,
                "rotary_append: bad cache sizes");
    VTX_REQUIRE(!tokens || ((!f.Hq || f.q_out) && p->v && p->k_pages && p->v_pages && p->block_table), VTX_ERR_BAD_ARG,
                "rotary_append: null pointer");
    VTX_REQUIRE(p->seq_ids || tokens <= p->num_seqs, VTX_ERR_BAD_ARG, "rotary_append: %lld tokens, %lld rows of the block table",
                (long long)tokens, (long long)p->num_seqs);
    a.r[1].dst = p->k_pages; a.r[1].db = p->k_stride_page; a.r[1].dl = p->k_stride_slot; a.r[1].dh = p->k_stride_head;
    a.r[2] = Rows{p->v, p->v_stride_b, p->v_stride_l, p->v_stride_h, p->v_pages, p->v_pages_stride_page, p->v_pages_stride_slot,
                  p->v_pages_stride_head, nullptr, 0, (int)f.Hk};
    a.paged = 1;
    a.table = p->block_table; a.table_stride = p->table_stride; a.table_width = p->table_width; a.seq_ids = p->seq_ids;
    a.num_seqs = p->num_seqs; a.num_pages = p->num_pages; a.page_size = p->page_size;
    return launch_fwd(a, f.io_dtype, (cudaStream_t)stream, "rotary_append");
}
