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
    float* dw_part;              // [blocks][2][D]
};

constexpr int kThreads = 256;
constexpr int kMaxD = 512;
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

template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    __device__ static void unpack(const uint4& v, float* f) {
        const T* p = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = to_f32<T>(p[i]);
    }
    __device__ static uint4 pack(const float* f) {
        uint4 v;
        T* p = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f32<T>(f[i]);
        return v;
    }
};

// Two vectors of N values turned in place: pairs (xa[i], xb[i]) in the half layout, neighbours in the interleaved one.
template <int N, bool INTER> __device__ __forceinline__ void rotate(float* xa, float* xb, const float2* cs) {
    if (INTER) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float a0 = xa[2 * i], a1 = xa[2 * i + 1], b0 = xb[2 * i], b1 = xb[2 * i + 1];
            const float2 p = cs[i], q = cs[N / 2 + i];
            xa[2 * i] = a0 * p.x - a1 * p.y; xa[2 * i + 1] = a0 * p.y + a1 * p.x;
            xb[2 * i] = b0 * q.x - b1 * q.y; xb[2 * i + 1] = b0 * q.y + b1 * q.x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = xa[i], y = xb[i];
            xa[i] = x * cs[i].x - y * cs[i].y; xb[i] = x * cs[i].y + y * cs[i].x;
        }
    }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What a thread of the vector kernels does in every row: two 16-byte vectors of a head, whose pairs are complete.
template <typename T, bool INTER> struct Lane {
    static constexpr int N = Vec<T>::N;
    int ea, eb;          // first elements of the two vectors
    bool on, turned;     // inside the head; inside its rotated part
    float2 cs[N];
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
    __device__ void load_turns(const float2* row, int sub) {
        if (turned)
#pragma unroll
            for (int i = 0; i < N; ++i) cs[i] = row[sub * N + i];
    }
};

// Block: `tb` tokens, 256 threads = rows of `lanes` threads (a power of two that covers a head); the rows of a token take its
// heads in turn.  Four heads' loads are issued before the first is used.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_fwd_kernel(const __grid_constant__ RotArgs a, int tb, int lane_shift) {
    constexpr int N = Vec<T>::N, U = 4;
    extern __shared__ float2 s_cs[];                               // [tb][rot / 2]
    __shared__ float s_w[2][kMaxD];
    __shared__ int64_t s_slot[8][2];
    const int tid = threadIdx.x, lanes = 1 << lane_shift, sub = tid & (lanes - 1), row = tid >> lane_shift;
    const int per_token = (kThreads >> lane_shift) / tb, ti = row / per_token, slot = row - ti * per_token;
    const int64_t T0 = (int64_t)blockIdx.x * tb, tokens = a.B * a.L;
    const int half = a.rot / 2;
    for (int i = tid; i < tb * half; i += kThreads) {
        const int t = i / half;
        const int64_t tok = T0 + t;
        if (tok < tokens) s_cs[i] = turn(a, load_pos(a, tok / a.L, tok % a.L), i - t * half);
    }
    for (int i = tid; i < 2 * a.D; i += kThreads) {
        const int which = i >= a.D;
        if (a.r[which].w) s_w[which][i - which * a.D] = ld_param(a.r[which].w, a.r[which].wd, i - which * a.D);
    }
    if (a.paged && tid < 2 * tb && T0 + tid / 2 < tokens)
        s_slot[tid / 2][tid & 1] = slot_offset(a, T0 + tid / 2, load_pos(a, (T0 + tid / 2) / a.L, (T0 + tid / 2) % a.L), 1 + (tid & 1));
    __syncthreads();
    Lane<T, INTER> ln(a, sub);
    const int64_t tok = T0 + ti;
    const bool live = ln.on && tok < tokens;
    if (live) ln.load_turns(s_cs + ti * half, sub);
    const int64_t b = live ? tok / a.L : 0, l = live ? tok - b * a.L : 0;
    const int heads = a.r[0].H + a.r[1].H + a.r[2].H;
    for (int h0 = 0; h0 < heads; h0 += per_token * U) {
        uint4 va[U], vb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int h = h0 + u * per_token + slot;
            va[u] = vb[u] = make_uint4(0, 0, 0, 0);
            if (live && h < heads) {
                const int which = h < a.r[0].H ? 0 : h < a.r[0].H + a.r[1].H ? 1 : 2;
                h -= which == 0 ? 0 : which == 1 ? a.r[0].H : a.r[0].H + a.r[1].H;
                const Rows& r = a.r[which];
                const T* p = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + h * r.sh;
                va[u] = *reinterpret_cast<const uint4*>(p + ln.ea);
                vb[u] = *reinterpret_cast<const uint4*>(p + ln.eb);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int h = h0 + u * per_token + slot;
            if (h0 + u * per_token >= heads) break;                // (the same for the whole block)
            const bool mine = live && h < heads;
            const int which = h < a.r[0].H ? 0 : h < a.r[0].H + a.r[1].H ? 1 : 2;
            h -= which == 0 ? 0 : which == 1 ? a.r[0].H : a.r[0].H + a.r[1].H;
            const Rows& r = a.r[which];
            float xa[N], xb[N];
            Vec<T>::unpack(va[u], xa);
            Vec<T>::unpack(vb[u], xb);
            if (a.r[0].w || a.r[1].w) {                            // (uniform: the lanes of a head meet)
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) ss += xa[i] * xa[i] + xb[i] * xb[i];
                ss = group_sum(ss, lanes);
                if (which < 2 && r.w && mine) {
                    const float inv = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        xa[i] *= inv * s_w[which][ln.ea + i];
                        xb[i] *= inv * s_w[which][ln.eb + i];
                    }
                }
            }
            if (!mine) continue;
            T* d = static_cast<T*>(r.dst) + h * r.dh;
            if (a.paged && which) {
                const int64_t at = s_slot[ti][which - 1];
                if (at < 0) continue;
                d += at;
            } else {
                d += b * r.db + l * r.dl;
            }
            if (which < 2) {
                if (ln.turned) rotate<N, INTER>(xa, xb, ln.cs);
                va[u] = Vec<T>::pack(xa);
                vb[u] = Vec<T>::pack(xb);
            }
            *reinterpret_cast<uint4*>(d + ln.ea) = va[u];
            *reinterpret_cast<uint4*>(d + ln.eb) = vb[u];
        }
    }
}

// Backward behind a norm.  The blocks walk the tokens; a thread keeps its dimensions through all rows, so the weights'
// gradients gather in its registers, then across the block's rows, and leave as one row of partial sums per block: summed in
// a fixed order, no atomics.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_bwd_kernel(const __grid_constant__ RotArgs a, int tb, int lane_shift) {
    constexpr int N = Vec<T>::N, U = 2;
    extern __shared__ float2 s_cs[];                               // [tb][rot / 2], later the rows' sums [rows][D]
    __shared__ float s_w[2][kMaxD];
    const int tid = threadIdx.x, lanes = 1 << lane_shift, sub = tid & (lanes - 1), row = tid >> lane_shift;
    const int rows = kThreads >> lane_shift, per_token = rows / tb, ti = row / per_token, slot = row - ti * per_token;
    const int64_t tokens = a.B * a.L;
    const int half = a.rot / 2;
    for (int i = tid; i < 2 * a.D; i += kThreads) {
        const int which = i >= a.D;
        s_w[which][i - which * a.D] = a.r[which].w ? ld_param(a.r[which].w, a.r[which].wd, i - which * a.D) : 1.f;
    }
    Lane<T, INTER> ln(a, sub);
    float dw[2][2 * N] = {};
    for (int64_t T0 = (int64_t)blockIdx.x * tb; T0 < tokens; T0 += (int64_t)gridDim.x * tb) {
        __syncthreads();
        for (int i = tid; i < tb * half; i += kThreads) {
            const int t = i / half;
            const int64_t tok = T0 + t;
            if (tok < tokens) s_cs[i] = turn(a, load_pos(a, tok / a.L, tok % a.L), i - t * half);
        }
        __syncthreads();
        const int64_t tok = T0 + ti;
        const bool live = ln.on && tok < tokens;
        if (live) ln.load_turns(s_cs + ti * half, sub);
        const int64_t b = live ? tok / a.L : 0, l = live ? tok - b * a.L : 0;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const Rows& r = a.r[which];
            for (int h0 = 0; h0 < r.H; h0 += per_token * U) {
                uint4 va[U], vb[U], ga[U], gb[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int h = h0 + u * per_token + slot;
                    va[u] = vb[u] = ga[u] = gb[u] = make_uint4(0, 0, 0, 0);
                    if (live && h < r.H) {
                        const T* p = static_cast<const T*>(r.src) + b * r.sb + l * r.sl + h * r.sh;
                        const T* g = static_cast<const T*>(a.dy[which]) + b * a.dyb[which] + l * a.dyl[which] + h * a.dyh[which];
                        va[u] = *reinterpret_cast<const uint4*>(p + ln.ea);
                        vb[u] = *reinterpret_cast<const uint4*>(p + ln.eb);
                        ga[u] = *reinterpret_cast<const uint4*>(g + ln.ea);
                        gb[u] = *reinterpret_cast<const uint4*>(g + ln.eb);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int h = h0 + u * per_token + slot;
                    float xa[N], xb[N], da[N], db[N];
                    Vec<T>::unpack(va[u], xa);
                    Vec<T>::unpack(vb[u], xb);
                    Vec<T>::unpack(ga[u], da);
                    Vec<T>::unpack(gb[u], db);
                    if (ln.turned) rotate<N, INTER>(da, db, ln.cs);
                    if (r.w) {
                        float ss = 0.f, dot = 0.f;
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            ss += xa[i] * xa[i] + xb[i] * xb[i];
                            dot += s_w[which][ln.on ? ln.ea + i : 0] * da[i] * xa[i] + s_w[which][ln.on ? ln.eb + i : 0] * db[i] * xb[i];
                        }
                        ss = group_sum(ss, lanes);
                        dot = group_sum(dot, lanes);
                        const float inv = rsqrtf(ss / (float)a.D + a.eps);
                        const float back = dot * inv * inv / (float)a.D;    // mean(w g xh) / r, to multiply x
                        if (live && h < r.H) {
#pragma unroll
                            for (int i = 0; i < N; ++i) {
                                dw[which][i] += da[i] * xa[i] * inv;
                                dw[which][N + i] += db[i] * xb[i] * inv;
                                da[i] = inv * (s_w[which][ln.ea + i] * da[i] - back * xa[i]);
                                db[i] = inv * (s_w[which][ln.eb + i] * db[i] - back * xb[i]);
                            }
                        }
                    }
                    if (live && h < r.H) {
                        T* d = static_cast<T*>(r.dst) + b * r.db + l * r.dl + h * r.dh;
                        *reinterpret_cast<uint4*>(d + ln.ea) = Vec<T>::pack(da);
                        *reinterpret_cast<uint4*>(d + ln.eb) = Vec<T>::pack(db);
                    }
                }
            }
        }
    }
    float* s_sum = reinterpret_cast<float*>(s_cs);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        if (ln.on)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s_sum[row * a.D + ln.ea + i] = dw[which][i];
                s_sum[row * a.D + ln.eb + i] = dw[which][N + i];
            }
        __syncthreads();
        for (int d = tid; d < a.D; d += kThreads) {
            float s = 0.f;
            for (int i = 0; i < rows; ++i) s += s_sum[i * a.D + d];
            a.dw_part[((int64_t)blockIdx.x * 2 + which) * a.D + d] = s;
        }
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
        float s = 0.f;
        for (int w = 0; w < warps; ++w) s += s_dw[(int64_t)w * 2 * a.D + i];
        a.dw_part[(int64_t)blockIdx.x * 2 * a.D + i] = s;
    }
}

// Partial sums [blocks][2][D] -> the two weight gradients, in the weights' types.  A warp per value.
__global__ void __launch_bounds__(kThreads) rotary_dw_kernel(const float* part, int blocks, int D, void* dwq, int qd, void* dwk, int kd) {
    const int i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= 2 * D) return;
    void* out = i < D ? dwq : dwk;
    if (!out) return;
    float s = 0.f;
    for (int b = lane; b < blocks; b += 32) s += part[(int64_t)b * 2 * D + i];
    s = group_sum(s, 32);
    if (lane) return;
    const int code = i < D ? qd : kd, at = i < D ? i : i - D;
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
    // one token per block until the blocks fill the machine several times over, then up to four
    int tb = tokens >= (int64_t)kNumSMs * 32 ? 4 : 1;
    tb = tb < (kThreads >> shift) ? tb : (kThreads >> shift);
    const int64_t blocks = ceil_div<int64_t>(tokens, tb);
    VTX_REQUIRE(blocks < ((int64_t)1 << 31), VTX_ERR_UNSUPPORTED, "%s: more than 2^31 tokens", who);
    const size_t smem = (size_t)tb * (a.rot / 2) * sizeof(float2);
    VTX_DISPATCH_IO(io, T, {
        if (a.inter) rotary_fwd_kernel<T, true><<<(unsigned)blocks, kThreads, smem, s>>>(a, tb, shift);
        else rotary_fwd_kernel<T, false><<<(unsigned)blocks, kThreads, smem, s>>>(a, tb, shift);
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
    int64_t blocks = 0;
    long long launches = 1;
    if (tokens && f.Hq + f.Hk) {
        const int shift = vector_lanes(a, dtype_size(f.io_dtype));
        launches = 2;
        if (shift < 0) {
            blocks = ceil_div<int64_t>(tokens * (f.Hq + f.Hk), kThreads / 32);
            blocks = blocks < kBwdBlocks ? blocks : kBwdBlocks;
            VTX_DISPATCH_IO(f.io_dtype, T,
                            rotary_bwd_any_kernel<T><<<(unsigned)blocks, kThreads, (size_t)(kThreads / 32) * 2 * f.D * 4, s>>>(a));
        } else {
            const int rows = kThreads >> shift;
            const int tb = rows < 4 ? rows : 4;
            blocks = ceil_div<int64_t>(tokens, tb);
            blocks = blocks < kBwdBlocks ? blocks : kBwdBlocks;
            size_t smem = (size_t)tb * (a.rot / 2) * sizeof(float2);
            const size_t sums = (size_t)rows * f.D * 4;
            smem = smem > sums ? smem : sums;
            VTX_DISPATCH_IO(f.io_dtype, T, {
                if (a.inter) rotary_bwd_kernel<T, true><<<(unsigned)blocks, kThreads, smem, s>>>(a, tb, shift);
                else rotary_bwd_kernel<T, false><<<(unsigned)blocks, kThreads, smem, s>>>(a, tb, shift);
            });
        }
    }
    rotary_dw_kernel<<<(unsigned)ceil_div<int64_t>(2 * f.D, kThreads / 32), kThreads, 0, s>>>(
        a.dw_part, (int)blocks, (int)f.D, f.q_weight ? p->dq_weight : nullptr, (int)f.q_weight_dtype,
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
