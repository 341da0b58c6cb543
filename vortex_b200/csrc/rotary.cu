// Rotary positions, optionally behind an RMS norm of each head, of the queries and keys of an attention layer; the same with
// the keys and values stored in the pages of a cache; and the backward pass.
//
//   xh = x / r, r = sqrt(mean_d x^2 + eps);  u = w * xh  (u = x without a weight);
//   pair i of the first `rot` dimensions turns by t_i = position * inv_freq[i]:
//     y_a = s (u_a cos t_i - u_b sin t_i),  y_b = s (u_a sin t_i + u_b cos t_i);  the other dimensions keep u.
//   backward, with g = the transposed rotation of dy:  dx = (w g - xh mean(w g xh)) / r,  dw = sum over rows of g xh.
//
// Every value is read once and written once, in fp32 between the two, rounded once: memory bounds it, and below some 10^4
// rows the launch.  What is shared is shared: the sine and cosine of a (token, pair) are formed once per block and token, in
// shared memory, and used by all heads.  The angle is formed in 64 bits, as turns with the whole turns taken off, since
// position * inv_freq in 32 bits is off by 0.03 rad at position 2^20; what is left goes to sincospif.
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
    float scale, eps;
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
constexpr int kFwdBlocks = 3, kFwdSteps = 2, kBwdPerSM = 2;
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

// Element offset of a token's row in the pages of the k (which = 1) or v (2) pool, or -1 where the token is not stored: a
// negative position is padding; one behind its table row, or a page outside the pool, sets the status word.
__device__ __forceinline__ int64_t slot_offset(const RotArgs& a, int64_t tok, int64_t pos, int which) {
    if (pos < 0) return -1;
    const int64_t seq = a.seq_ids ? (int64_t)a.seq_ids[tok] : tok;
    const int64_t at = pos / a.page_size;
    int64_t page = -1;
    if (seq >= 0 && seq < a.num_seqs && at < a.table_width) page = a.table[seq * a.table_stride + at];
    if (page < 0 || page >= a.num_pages) {
        atomicCAS(&g_device_status, 0, kStatusBadPage);
        return -1;
    }
    return page * a.r[which].db + (pos - at * a.page_size) * a.r[which].dl;
}

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
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    T t[2] = {from_f32<T>(lo), from_f32<T>(hi)};
    return *reinterpret_cast<uint32_t*>(t);
}
__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
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
    f32x2 c[P], s[P];
    __device__ Lane(const RotArgs& a, int sub) {
        on = sub * 2 * N < a.D;
        turned = sub * 2 * N < a.rot;
        if (INTER) {
            ea = sub * 2 * N; eb = ea + N;
        } else if (turned) {
            ea = sub * N; eb = ea + a.rot / 2;
        } else {                                     // the kept part is halved like the turned one
            ea = a.rot + (sub * 2 * N - a.rot) / 2; eb = ea + (a.D - a.rot) / 2;
        }
    }
    // element of the head that value i of the 2N holds (a first, then b)
    __device__ int element(int i) const { return INTER ? ea + 2 * (i < N ? i : i - N) + (i >= N) : i < N ? ea + i : eb + i - N; }
    // cosines of a token's pairs, then their sines
    __device__ void load_turns(const float* turns, int half, int sub) {
        if (!turned) return;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            c[i] = *reinterpret_cast<const f32x2*>(turns + sub * N + 2 * i);
            s[i] = *reinterpret_cast<const f32x2*>(turns + half + sub * N + 2 * i);
        }
    }
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
    __device__ void rotate(f32x2* a, f32x2* b) const {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const f32x2 x = a[i], y = b[i];
            a[i] = sub2(mul2(x, c[i]), mul2(y, s[i]));
            b[i] = fma2(x, s[i], mul2(y, c[i]));
        }
    }
};

// The weights as the lanes hold them, in shared memory: quad q of a lane's 2N values at [q][lane], so that the lanes of a head
// read neighbouring 16 bytes.
template <typename T, bool INTER> __device__ __forceinline__ void stage_weights(const RotArgs& a, const Rows& r, float* dst, int lanes) {
    constexpr int N = Lane<T, INTER>::N;
    for (int i = threadIdx.x; i < 2 * N * lanes; i += kThreads) {
        const int q = i / (4 * lanes), sub = i / 4 - q * lanes;
        const Lane<T, INTER> ln(a, sub);
        dst[i] = ln.on && r.w ? ld_param(r.w, r.wd, ln.element(q * 4 + (i & 3))) : 1.f;
    }
}
__device__ __forceinline__ void load_quad(const float* w, int q, int lanes, int sub, f32x2& w0, f32x2& w1) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(w + (q * lanes + sub) * 4);
    w0 = v.x;
    w1 = v.y;
}

// Cosines and sines of a token's pairs, in the warp's piece of shared memory.
__device__ __forceinline__ void warp_turns(const RotArgs& a, float* mine, int64_t pos) {
    const int half = a.rot / 2;
    __syncwarp();
    for (int i = threadIdx.x & 31; i < half; i += 32) {
        const float2 cs = turn(a, pos, i);
        mine[i] = cs.x;
        mine[half + i] = cs.y;
    }
    __syncwarp();
}

// A warp takes one token and `chunk` heads of its queries, keys or values, 32 >> lane_shift heads side by side
// (1 << lane_shift lanes cover a head), U steps in flight: a step's registers are refilled as soon as its values have been
// unpacked.  No warp waits for another (but for the weights, once): a token's chain position -> angles, page lookup -> store
// hides behind the other warps' traffic.
struct Chunks { int size, q, k, v; };      // heads in one; chunks of a token's queries, keys, values

template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads, kFwdBlocks) rotary_fwd_kernel(const __grid_constant__ RotArgs a, Chunks ch, int lane_shift) {
    using Ln = Lane<T, INTER>;
    constexpr int N = Ln::N, P = Ln::P, U = kFwdSteps;
    extern __shared__ __align__(16) float s_turn[];                // [warp][rot]
    __shared__ __align__(16) float s_w[2][kMaxD];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lanes = 1 << lane_shift, sub = lane & (lanes - 1), slot = lane >> lane_shift;
    const int step = 32 >> lane_shift;
    const bool any_norm = a.r[0].w || a.r[1].w;
    const uint32_t item = blockIdx.x * (kThreads / 32) + warp, per = ch.q + ch.k + ch.v, tok = item / per, L = (uint32_t)a.L;
    const bool live = tok < (uint32_t)(a.B * a.L);
    int c = (int)(item - tok * per);
    const int which = c < ch.q ? 0 : c < ch.q + ch.k ? 1 : 2;
    c -= which == 0 ? 0 : which == 1 ? ch.q : ch.q + ch.k;
    const Rows& r = a.r[which];
    const uint32_t b = live ? tok / L : 0, l = live ? tok - b * L : 0;
    const int first = c * ch.size, count = live ? (ch.size < r.H - first ? ch.size : r.H - first) : 0;
    Ln ln(a, sub);
    const T* src = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + (first + slot) * r.sh;
    const int64_t src_step = step * r.sh;
    uint4 va[U], vb[U];
    int fh = slot;                                                 // head of the next step to fetch
    auto fetch = [&](int u) {
        va[u] = vb[u] = make_uint4(0, 0, 0, 0);
        if (ln.on && fh < count) {
            va[u] = *reinterpret_cast<const uint4*>(src + ln.ea);
            vb[u] = *reinterpret_cast<const uint4*>(src + ln.eb);
        }
        src += src_step;
        fh += step;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(u);
    if (any_norm) {
        stage_weights<T, INTER>(a, a.r[0], s_w[0], lanes);
        stage_weights<T, INTER>(a, a.r[1], s_w[1], lanes);
        __syncthreads();
    }
    if (!live) return;
    const int64_t pos = load_pos(a, b, l);
    int64_t at = b * r.db + l * r.dl;
    if (a.paged && which) {
        at = slot_offset(a, tok, pos, which);
        if (at < 0) return;
    }
    T* dst = static_cast<T*>(r.dst) + at + (first + slot) * r.dh;
    const int64_t dst_step = step * r.dh;
    if (which < 2) {
        warp_turns(a, s_turn + warp * a.rot, pos);
        ln.load_turns(s_turn + warp * a.rot, a.rot / 2, sub);
    }
    const bool norm = which < 2 && r.w;
    for (int h0 = 0; h0 < count;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h0 >= count) break;                                // (the same for the whole warp)
            const bool mine = ln.on && h0 + slot < count;
            uint4 ra = va[u], rb = vb[u];
            fetch(u);
            if (which < 2) {
                f32x2 xa[P], xb[P];
                Ln::unpack(ra, rb, xa, xb);
                if (norm) {
                    f32x2 ss2 = mul2(xa[0], xa[0]);
#pragma unroll
                    for (int i = 1; i < P; ++i) ss2 = fma2(xa[i], xa[i], ss2);
#pragma unroll
                    for (int i = 0; i < P; ++i) ss2 = fma2(xb[i], xb[i], ss2);
                    const float ss = group_sum(sum2(ss2), lanes);
                    const float inv = rsqrtf(ss / (float)a.D + a.eps);
                    const f32x2 inv2 = pk2(inv, inv);
#pragma unroll
                    for (int q = 0; q < N / 2; ++q) {
                        f32x2 w0, w1;
                        load_quad(s_w[which], q, lanes, sub, w0, w1);
                        f32x2* x = q < N / 4 ? xa + 2 * q : xb + 2 * (q - N / 4);
                        x[0] = mul2(mul2(x[0], inv2), w0);
                        x[1] = mul2(mul2(x[1], inv2), w1);
                    }
                }
                if (ln.turned) ln.rotate(xa, xb);
                Ln::pack(xa, xb, ra, rb);
            }
            if (mine) {
                *reinterpret_cast<uint4*>(dst + ln.ea) = ra;
                *reinterpret_cast<uint4*>(dst + ln.eb) = rb;
            }
            dst += dst_step;
            h0 += step;
        }
    }
}

// Backward behind a norm.  The first blocks take the queries, the rest the keys; a warp walks its tokens, all heads of one
// before the next, U steps in flight across them.  A lane keeps its dimensions through all rows, so the weight's gradient
// gathers in its registers, then across the block, and leaves as one row of partial sums per block: summed in a fixed order,
// no atomics.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads, kBwdPerSM) rotary_bwd_kernel(const __grid_constant__ RotArgs a, int q_blocks, int lane_shift) {
    using Ln = Lane<T, INTER>;
    constexpr int N = Ln::N, P = Ln::P, U = 2;
    extern __shared__ __align__(16) float s_turn[];                // [warp][rot], later the rows' sums [rows][D]
    __shared__ __align__(16) float s_w[kMaxD];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lanes = 1 << lane_shift, sub = lane & (lanes - 1), slot = lane >> lane_shift;
    const int step = 32 >> lane_shift, rows = kThreads >> lane_shift;
    const int which = (int)blockIdx.x >= q_blocks;
    const Rows& r = a.r[which];
    const uint32_t tokens = (uint32_t)(a.B * a.L), L = (uint32_t)a.L;
    const uint32_t w0 = (blockIdx.x - (which ? q_blocks : 0)) * (kThreads / 32) + warp;
    const uint32_t warps = (which ? gridDim.x - q_blocks : q_blocks) * (kThreads / 32);
    const bool norm = r.w;
    Ln ln(a, sub);
    f32x2 dwa[P], dwb[P];
#pragma unroll
    for (int i = 0; i < P; ++i) dwa[i] = dwb[i] = pk2(0.f, 0.f);
    uint4 va[U], vb[U], ga[U], gb[U];
    uint32_t ft = w0;                                              // token and first head of the next step to fetch
    int fh = 0;
    const T *xp = nullptr, *gp = nullptr;
    const int64_t xstep = step * r.sh, gstep = step * a.dyh[which];
    auto fetch = [&](int u) {
        va[u] = vb[u] = ga[u] = gb[u] = make_uint4(0, 0, 0, 0);
        if (fh == 0) {
            const uint32_t b = ft / L, l = ft - b * L;
            xp = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + slot * r.sh;
            gp = static_cast<const T*>(a.dy[which]) + b * a.dyb[which] + l * a.dyl[which] + slot * a.dyh[which];
        }
        if (ln.on && ft < tokens && fh + slot < r.H) {
            ga[u] = *reinterpret_cast<const uint4*>(gp + ln.ea);
            gb[u] = *reinterpret_cast<const uint4*>(gp + ln.eb);
            if (norm) {
                va[u] = *reinterpret_cast<const uint4*>(xp + ln.ea);
                vb[u] = *reinterpret_cast<const uint4*>(xp + ln.eb);
            }
        }
        xp += xstep;
        gp += gstep;
        fh += step;
        if (fh >= r.H) { fh = 0; ft = ft + warps < ft ? tokens : ft + warps; }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(u);
    stage_weights<T, INTER>(a, r, s_w, lanes);
    __syncthreads();
    uint32_t t = w0;
    int h0 = 0;
    T* dst = nullptr;
    const int64_t dstep = step * r.dh;
    while (t < tokens) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t >= tokens) break;
            if (h0 == 0) {
                const uint32_t b = t / L, l = t - b * L;
                warp_turns(a, s_turn + warp * a.rot, load_pos(a, b, l));
                ln.load_turns(s_turn + warp * a.rot, a.rot / 2, sub);
                dst = static_cast<T*>(r.dst) + b * r.db + l * r.dl + slot * r.dh;
            }
            f32x2 xa[P], xb[P], da[P], db[P];
            Ln::unpack(va[u], vb[u], xa, xb);
            Ln::unpack(ga[u], gb[u], da, db);
            fetch(u);
            if (ln.turned) ln.rotate(da, db);
            if (norm) {
                f32x2 ss2 = mul2(xa[0], xa[0]), dot2 = pk2(0.f, 0.f);
#pragma unroll
                for (int i = 1; i < P; ++i) ss2 = fma2(xa[i], xa[i], ss2);
#pragma unroll
                for (int i = 0; i < P; ++i) ss2 = fma2(xb[i], xb[i], ss2);
                const float ss = group_sum(sum2(ss2), lanes);
                const float inv = rsqrtf(ss / (float)a.D + a.eps);
                const f32x2 inv2 = pk2(inv, inv);
#pragma unroll
                for (int q = 0; q < N / 2; ++q) {
                    f32x2 wq[2];
                    load_quad(s_w, q, lanes, sub, wq[0], wq[1]);
                    const int at = q < N / 4 ? 2 * q : 2 * (q - N / 4);
                    f32x2 *x = (q < N / 4 ? xa : xb) + at, *d = (q < N / 4 ? da : db) + at, *dw = (q < N / 4 ? dwa : dwb) + at;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // (lanes outside the head and its rows hold zeros)
                        x[j] = mul2(x[j], inv2);                            // xh
                        dw[j] = fma2(d[j], x[j], dw[j]);
                        d[j] = mul2(d[j], wq[j]);                           // w g
                        dot2 = fma2(d[j], x[j], dot2);
                    }
                }
                const float mean = group_sum(sum2(dot2), lanes) * (-1.f / (float)a.D);
                const f32x2 mean2 = pk2(mean, mean);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    da[i] = mul2(fma2(mean2, xa[i], da[i]), inv2);
                    db[i] = mul2(fma2(mean2, xb[i], db[i]), inv2);
                }
            }
            if (ln.on && h0 + slot < r.H) {
                uint4 ra, rb;
                Ln::pack(da, db, ra, rb);
                *reinterpret_cast<uint4*>(dst + ln.ea) = ra;
                *reinterpret_cast<uint4*>(dst + ln.eb) = rb;
            }
            dst += dstep;
            h0 += step;
            if (h0 >= r.H) { h0 = 0; t = t + warps < t ? tokens : t + warps; }
        }
    }
    float* s_sum = s_turn;
    const int row = tid >> lane_shift;
    __syncthreads();
    if (ln.on)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float lo, hi;
            up2(dwa[i / 2], lo, hi);
            s_sum[row * a.D + ln.element(i)] = i & 1 ? hi : lo;
            up2(dwb[i / 2], lo, hi);
            s_sum[row * a.D + ln.element(N + i)] = i & 1 ? hi : lo;
        }
    __syncthreads();
    for (int d = tid; d < a.D; d += kThreads) {
        float sum = 0.f;
        for (int i = 0; i < rows; ++i) sum += s_sum[i * a.D + d];
        a.dw_part[(int64_t)blockIdx.x * a.D + d] = sum;
    }
}

// Any head size and alignment: a warp per (token, head), values one by one.  Pair i, and the kept dimensions behind the
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
        const int64_t at = slot_offset(a, tok, pos, which);
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
        inv = rsqrtf(group_sum(ss, 32) / (float)a.D + a.eps);
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
                inv = rsqrtf(group_sum(ss, 32) / (float)a.D + a.eps);
                back = group_sum(dot, 32) * inv * inv / (float)a.D;
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

// Partial sums, q_rows rows of D for the queries and k_rows for the keys, -> the two weight gradients in the weights' types.  A
// warp per value.
__global__ void __launch_bounds__(kThreads) rotary_dw_kernel(const float* part, int q_rows, int k_rows, int D, void* dwq, int qd, void* dwk, int kd) {
    const int i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= 2 * D) return;
    const bool key = i >= D;
    void* out = key ? dwk : dwq;
    if (!out) return;
    const int at = key ? i - D : i, rows = key ? k_rows : q_rows;
    const float* p = part + (key ? (int64_t)q_rows * D : 0) + at;
    float s = 0.f;
    for (int b = lane; b < rows; b += 32) s += p[(int64_t)b * D];
    s = group_sum(s, 32);
    if (lane) return;
    const int code = key ? kd : qd;
    if (code == VTX_F32) static_cast<float*>(out)[at] = s;
    else if (code == VTX_BF16) static_cast<__nv_bfloat16*>(out)[at] = from_f32<__nv_bfloat16>(s);
    else static_cast<__half*>(out)[at] = from_f32<__half>(s);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
bool rows_aligned(const void* p, int64_t sb, int64_t sl, int64_t sh, int64_t es) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (sb * es) % 16 == 0 && (sl * es) % 16 == 0 && (sh * es) % 16 == 0;
}

// Lanes of a head in the vector kernels, as a shift; -1 where they do not apply: heads and their rotated part in whole pairs
// of 16-byte vectors, at most 32 threads to a head, all rows on 16-byte boundaries.
int vector_lanes(const RotArgs& a, int64_t es) {
    const int pair = 2 * (int)(16 / es);
    if (a.D % pair || a.rot % pair || a.D / pair > 32) return -1;
    for (int i = 0; i < 3; ++i) {
        const Rows& r = a.r[i];
        if (r.H && (!rows_aligned(r.src, r.sb, r.sl, r.sh, es) || !rows_aligned(r.dst, r.db, r.dl, r.dh, es))) return -1;
        if (i < 2 && r.H && a.dy[i] && !rows_aligned(a.dy[i], a.dyb[i], a.dyl[i], a.dyh[i], es)) return -1;
    }
    int shift = 0;
    while ((1 << shift) * pair < a.D) ++shift;
    return shift;
}

int launch_fwd(const RotArgs& a, int64_t io, cudaStream_t s, const char* who) {
    const int64_t tokens = a.B * a.L, heads = a.r[0].H + a.r[1].H + a.r[2].H;
    if (tokens == 0 || heads == 0) return VTX_OK;
    const int shift = vector_lanes(a, dtype_size(io));
    if (shift < 0) {
        const int64_t blocks = ceil_div<int64_t>(tokens * heads, kThreads / 32);
        VTX_REQUIRE(blocks < ((int64_t)1 << 31), VTX_ERR_UNSUPPORTED, "%s: more than 2^34 rows", who);
        VTX_DISPATCH_IO(io, T, rotary_fwd_any_kernel<T><<<(unsigned)blocks, kThreads, 0, s>>>(a));
        return check_launch(who);
    }
    // up to eight steps a warp once that still gives every SM its warps; below, fewer, down to one
    const int step = 32 >> shift;
    int steps = 8;
    auto chunks = [&](int h) { return (int)ceil_div<int64_t>(h, steps * step); };
    auto per_token = [&] { return (int64_t)chunks(a.r[0].H) + chunks(a.r[1].H) + chunks(a.r[2].H); };
    while (steps > 1 && tokens * per_token() < (int64_t)kNumSMs * kFwdBlocks * (kThreads / 32)) steps /= 2;
    const Chunks ch{steps * step, chunks(a.r[0].H), chunks(a.r[1].H), chunks(a.r[2].H)};
    const int64_t items = tokens * per_token(), blocks = ceil_div<int64_t>(items, kThreads / 32);
    VTX_REQUIRE(items < ((int64_t)1 << 32) - kThreads, VTX_ERR_UNSUPPORTED, "%s: more than 2^32 pieces of heads", who);
    const size_t smem = (size_t)(kThreads / 32) * a.rot * sizeof(float);
    VTX_DISPATCH_IO(io, T, {
        if (a.inter) rotary_fwd_kernel<T, true><<<(unsigned)blocks, kThreads, smem, s>>>(a, ch, shift);
        else rotary_fwd_kernel<T, false><<<(unsigned)blocks, kThreads, smem, s>>>(a, ch, shift);
    });
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
    a.B = p.B; a.L = p.L; a.D = (int)p.D;
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
    long long launches = 1;
    if (tokens && f.Hq + f.Hk) {
        const int shift = vector_lanes(a, dtype_size(f.io_dtype));
        launches = 2;
        if (shift < 0) {
            const int64_t warps = ceil_div<int64_t>(tokens * (f.Hq + f.Hk), kThreads / 32);
            q_rows = k_rows = warps < kBwdBlocks ? warps : kBwdBlocks;
            VTX_DISPATCH_IO(f.io_dtype, T,
                            rotary_bwd_any_kernel<T><<<(unsigned)q_rows, kThreads, (size_t)(kThreads / 32) * 2 * f.D * 4, s>>>(a));
        } else {
            // blocks for queries and keys in proportion to their heads, a warp at least a token
            const int64_t most = ceil_div<int64_t>(tokens, kThreads / 32), total = kNumSMs * kBwdPerSM;
            q_rows = f.Hq ? (total * f.Hq + (f.Hq + f.Hk) / 2) / (f.Hq + f.Hk) : 0;
            if (f.Hq) q_rows = q_rows < 1 ? 1 : f.Hk && q_rows > total - 1 ? total - 1 : q_rows;
            k_rows = f.Hk ? total - q_rows : 0;
            q_rows = q_rows < most ? q_rows : most;
            k_rows = k_rows < most ? k_rows : most;
            size_t smem = (size_t)(kThreads / 32) * a.rot * sizeof(float);
            const size_t sums = (size_t)(kThreads >> shift) * f.D * 4;
            smem = smem > sums ? smem : sums;
            const unsigned blocks = (unsigned)(q_rows + k_rows);
            VTX_DISPATCH_IO(f.io_dtype, T, {
                if (a.inter) rotary_bwd_kernel<T, true><<<blocks, kThreads, smem, s>>>(a, (int)q_rows, shift);
                else rotary_bwd_kernel<T, false><<<blocks, kThreads, smem, s>>>(a, (int)q_rows, shift);
            });
        }
    }
    rotary_dw_kernel<<<(unsigned)ceil_div<int64_t>(2 * f.D, kThreads / 32), kThreads, 0, s>>>(
        a.dw_part, (int)q_rows, (int)k_rows, (int)f.D, f.q_weight ? p->dq_weight : nullptr, (int)f.q_weight_dtype,
        f.k_weight ? p->dk_weight : nullptr, (int)f.k_weight_dtype);
    return check_launch("qk_norm_rotary_bwd", launches);
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
