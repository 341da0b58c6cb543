// Attention of one new token per sequence over a cache of keys and values in pages.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp2(s_j - m),  s_j = log2(e) * softmax_scale * (q . k_j)
//
// in one pass over the cache with a running maximum m.  Every key and value is read once for up to 16 query heads (8 where a head
// has more than 128 values, 4 on the CUDA cores; beyond, a pass over the cache for each so many), two operations a byte and head:
// memory bounds it.  Measured (bf16, of the measured copy bandwidth, replayed from a graph; in brackets as a program's calls on
// changing inputs): 64 sequences of 8192-8704 keys, 32 heads of 128, 1280-1318 us (1.0; 1405, 0.96) and one of 1,048,576 keys, 8
// heads, 640-666 us (1.0; 682, 0.96); 32 sequences of 4000-8000 keys, 64 query heads over 8, 130 us (0.93); 48 ragged ones, 32
// over 8 heads of 64 in fp16, 224-236 us (0.88-0.93; 254, 0.82); one of 700 keys 8.8 us (11.6; a chain of launch, lengths, table,
// keys, join and join's launch).  What the kernels are built around:
//
// * Work.  The cache is cut into units of 64 or 128 keys of one key head; the units of all sequences, in a row, are dealt out in
//   equal runs, whatever the lengths (they are on the device: every block sums them up itself), a run to a block for each head,
//   or, with the heads' units in the row as well, to one block (make_plan chooses).  A block's run covers the end of one
//   (sequence, head), some whole ones, and the beginning of another; whole ones are finished in place, the two open ones leave
//   (m, sum, unnormalised out) in the scratch, which the second kernel joins.  At most two open ones a block, and no
//   more blocks than the GPU runs at a time: the scratch grows with the work only as long as that has fewer units.  The second kernel is launched so that it is set up while the first still runs.
// * No shared memory on the way.  With keys as the rows of the first product (S^T = K Q^T) a lane's piece of the A operand is
//   16 contiguous bytes of two key rows, once the order of the summed dimensions is agreed with Q; for the second
//   (O^T = V^T P^T) it is 16 contiguous bytes of four value rows, after one byte permutation a register.  So loads go from
//   global memory to the registers that the mma.sync reads; 16 keys are 16 loads of 16 bytes a lane, the next tile's keys are
//   in flight from the moment the scores exist, its values from the moment the second product is issued.  Tensor cores at
//   16 x 8 x 16 are enough: with one query head of eight columns used their pipe is 15 % busy.
// * P is brought from the accumulator's layout to the B operand's by transposing 8 x 8 blocks (movmatrix), as head and
//   remainder: rounded to bf16 alone it would cost as much as the output's own rounding.
// * The maximum is raised only when a score passes it by more than a slack (2^8, for fp16 2^4): most tiles then need neither
//   the reduction over the lanes nor the rescaling; the sums stay below 2^15 * keys, far inside fp32.
#include <cfloat>

#include "attn.cuh"
#include "tma.cuh"
#include "umma.cuh"

VTX_DEFINE_STATUS_READER()

namespace vtx {
namespace {

constexpr int kThreads = 128, kWarps = 4, kTile = 16;
// Tiles of 16 keys that a warp has in flight together: two of the smaller heads are as many bytes as one of the larger.
constexpr int tiles(int DP) { return DP == 64 ? 2 : 1; }
// Keys of a unit of work, in the tensor-core kernel and in the other.
constexpr int unit_keys(int DP, bool tensor) { return kWarps * kTile * (tensor ? tiles(DP) : 1); }
// Reference m of a running sum: p = exp2(s - m).  The largest score seen stays between m + shift and m + shift + slack.
// fp16 keeps nothing below 2^-25: its probabilities are held near the top of its range (at most 2^15), so that even 2^20 keys
// of 2^-25 of the largest one's weight still count; bf16 and fp32 need no shift.
template <typename T> struct Ref {
    static constexpr bool half = DTypeCode<T>::value == VTX_F16;
    static constexpr float shift = half ? 11.f : 0.f, slack = half ? 4.f : 8.f;
};

struct AttnArgs {
    const void* q;
    int64_t qsb, qsh;
    const void* k;
    int64_t ksp, kss, ksh;
    const void* v;
    int64_t vsp, vss, vsh;
    const int32_t* table;           // NULL: page b is sequence b's
    int64_t ts;
    const int32_t* lens;
    void* out;
    int64_t osb, osh;
    float* lse;
    float* part;                    // [blocks][2][heads of a pass] rows of (DP sums)
    float2* part_ml;                // the same, (m, l)
    struct Open* open;              // [blocks]
    float scale;                    // log2(e) * softmax_scale
    int window;                     // INT_MAX: none
    int B, Hq, G, D, page_size, num_pages;
    int passes, head_groups;        // passes over the G query heads of a key head; Hk * passes
    int unit;                       // keys of a unit of work
    int abreast;                    // head groups whose blocks walk the same keys side by side (1, or all of them)
    int64_t max_keys;
};

// The (sequence, head group) that begins in a block's run and ends in the `runs`-th run from there.
struct Open {
    int64_t units;                  // of all runs
    int b, hg, runs, pad;
};

struct Seq {                        // keys lo .. n-1 of a sequence; tiles start at lo & ~15
    int lo, n, base, units;
    __device__ Seq(const AttnArgs& a, int b) {
        const int len = a.lens[b];
        n = len < 0 ? 0 : len;
        if (n > a.max_keys) {
            atomicCAS(&g_device_status, 0, kStatusBadPage);
            n = (int)a.max_keys;
        }
        lo = (len > a.window) ? len - a.window : 0;
        if (lo > n) lo = n;
        base = lo & ~(kTile - 1);
        units = n > base ? (int)(((unsigned)(n - base) + a.unit - 1) / a.unit) : 1;      // an empty one has a unit, to write its zeros
    }
};

// What comes out where a sequence and head ends with a sum of 0: zeros where no key was taken (none is counted, or the table gives
// none a page), and 0 / 0 where the scores of all that were are -inf.  Rare enough to look the pages up again, in a function of
// its own, so that the loops keep their registers.  (A flag kept beside the sums took 4 % of 64 query heads over 4; the lookup
// inlined at a piece's end, 12 % of fp16 heads of 64.)
__device__ __noinline__ float zero_sum(const AttnArgs& a, int b, int lo, int n) {
    if (lo >= n) return 0.f;
    if (!a.table) return NAN;
    for (int64_t i = lo / a.page_size; i <= (n - 1) / a.page_size; ++i) {
        const int page = a.table[b * a.ts + i];
        if (page >= 0 && page < a.num_pages) return NAN;
    }
    return 0.f;
}

__device__ __forceinline__ int64_t run_start(int64_t units, int w, int W) { return units * w / W; }

__device__ __forceinline__ int64_t warp_scan(int64_t v) {
    const int lane = threadIdx.x & 31;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// Inclusive sum over the block's threads, and the block's total.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s_tot, int64_t& total) {
    v = warp_scan(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 31) s_tot[threadIdx.x >> 5] = v;
    __syncthreads();
    total = 0;
    int64_t before = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < (int)(threadIdx.x >> 5)) before += s_tot[w];
        total += s_tot[w];
    }
    return v + before;
}

// The block's run of units and the sequence in which it starts.
struct Run {
    int64_t units, at, end, seq_first;     // of all; next, end; first unit of sequence b
    int b, hg0, inner, run, runs;          // sequence; the block's head group, or the first; head groups in the run; run of runs
    __device__ Run(const AttnArgs& a) {
        __shared__ int64_t s_tot[kWarps], s_first;
        __shared__ int s_b;
        const int tid = threadIdx.x;
        inner = a.head_groups / a.abreast;
        run = blockIdx.x / a.abreast;
        runs = gridDim.x / a.abreast;
        hg0 = blockIdx.x - run * a.abreast;
        if (a.B <= 32) {                    // every warp for itself
            const int lane = tid & 31;
            const int64_t own = lane < a.B ? (int64_t)Seq(a, lane).units * inner : 0, incl = warp_scan(own);
            units = __shfl_sync(0xffffffffu, incl, 31);
            at = run_start(units, run, runs);
            end = run_start(units, run + 1, runs);
            const unsigned in = __ballot_sync(0xffffffffu, at >= incl - own && at < incl);
            b = in ? __ffs(in) - 1 : 0;
            seq_first = __shfl_sync(0xffffffffu, incl - own, b);
            return;
        }
        int64_t mine = tid < a.B ? (int64_t)Seq(a, tid).units * inner : 0, total, incl;
        incl = block_scan(mine, s_tot, total);
        units = total;
        for (int c = kThreads; c < a.B; c += kThreads) {
            int64_t t;
            block_scan(c + tid < a.B ? (int64_t)Seq(a, c + tid).units * inner : 0, s_tot, t);
            units += t;
        }
        at = run_start(units, run, runs);
        end = run_start(units, run + 1, runs);
        int64_t before = 0;
        for (int c = 0;; c += kThreads) {
            if (c) {
                mine = c + tid < a.B ? (int64_t)Seq(a, c + tid).units * inner : 0;
                incl = block_scan(mine, s_tot, total);
            }
            if (at < before + total || c + kThreads >= a.B) {
                const int64_t first = before + incl - mine;
                if (at >= first && at < first + mine) { s_b = c + tid; s_first = first; }
                break;
            }
            before += total;
        }
        __syncthreads();
        b = s_b;
        seq_first = s_first;
    }
};

// One piece of work: units c0 .. c1-1 of a sequence and head group.
struct Piece {
    int b, hg, c0, c1, units, lo, n, base;
    int kvh, h0, heads;                    // key head, first query head, query heads
};

template <int HP> __device__ __forceinline__ Piece next_piece(const AttnArgs& a, Run& r) {
    const Seq s(a, r.b);
    Piece p;
    p.b = r.b; p.units = s.units; p.lo = s.lo; p.n = s.n; p.base = s.base;
    const int64_t in = r.at - r.seq_first;
    const int hg = (int)(in / s.units);
    p.hg = r.hg0 + hg;
    p.c0 = (int)(in - (int64_t)hg * s.units);
    const int64_t left = r.end - r.at;
    p.c1 = (int)(p.c0 + left < s.units ? p.c0 + left : s.units);
    p.kvh = p.hg / a.passes;
    const int first = (p.hg - p.kvh * a.passes) * HP;
    p.h0 = p.kvh * a.G + first;
    p.heads = a.G - first < HP ? a.G - first : HP;
    r.at += p.c1 - p.c0;
    if (hg == r.inner - 1 && p.c1 == s.units) {
        r.seq_first += (int64_t)s.units * r.inner;
        ++r.b;
    }
    return p;
}

// The warps' (m, l, out) of a piece, in shared memory, joined: a whole (sequence, head group) is finished, an open one stored.
template <typename T, int DP, int HP, int PITCH>
__device__ __forceinline__ void join_warps(const AttnArgs& a, const Piece& p, const Run& r, const float* s_o, const float (*s_m)[HP],
                                           const float (*s_l)[HP], bool vec) {
    const bool whole = p.c0 == 0 && p.c1 == p.units;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (p.c0 == 0);
    for (int i = threadIdx.x; i < p.heads * (DP / 4); i += kThreads) {
        const int h = i / (DP / 4), d = (i - h * (DP / 4)) * 4;
        float m = s_m[0][h];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w][h]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(s_m[w][h] - m);
            const float4 x = *reinterpret_cast<const float4*>(s_o + (w * HP + h) * PITCH + d);
            o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
            l += f * s_l[w][h];
        }
        if (whole) {
            const float f = l == 0.f ? zero_sum(a, p.b, p.lo, p.n) : 1.f / l;
            T* y = static_cast<T*>(a.out) + p.b * a.osb + (p.h0 + h) * a.osh + d;
            const float v[4] = {o.x * f, o.y * f, o.z * f, o.w * f};
            if (vec && d + 4 <= a.D) {
                T t[4];
                for (int j = 0; j < 4; ++j) t[j] = from_f32<T>(v[j]);
                if (sizeof(T) == 2) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<uint2*>(t);
                else *reinterpret_cast<uint4*>(y) = *reinterpret_cast<uint4*>(t);
            } else {
                for (int j = 0; j < 4; ++j) if (d + j < a.D) y[j] = from_f32<T>(v[j]);
            }
            if (d == 0 && a.lse) a.lse[(int64_t)p.b * a.Hq + p.h0 + h] = (m + log2f(l)) * 0.69314718055994531f;
        } else {
            *reinterpret_cast<float4*>(a.part + (slot * HP + h) * DP + d) = o;
            if (d == 0) a.part_ml[slot * HP + h] = make_float2(m, l);
        }
    }
    if (threadIdx.x == 0 && p.c0 == 0 && !whole) {
        const int64_t last_unit = r.at - p.c1 + p.units - 1;        // (r.at is behind this piece)
        int w = (int)(last_unit * r.runs / r.units);
        while (w + 1 < r.runs && run_start(r.units, w + 1, r.runs) <= last_unit) ++w;
        while (run_start(r.units, w, r.runs) > last_unit) --w;
        a.open[blockIdx.x] = Open{r.units, p.b, p.hg, w - r.run + 1, 0};
    }
}

// ---- tensor cores: 16-bit caches on 16-byte boundaries, heads of up to 256 values in eights --------------------------------
template <typename T> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 ld16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// Two probabilities p, q >= 0 as heads and remainders of the I/O type, packed: the head towards zero, so that no remainder is
// negative, and no remainder of a probability above the type's smallest step is zero: a value of infinity then comes out as
// infinity, not as the difference of two or as 0 * inf.  What that adds is below 2^-24 of the largest probability a key in
// fp16 (p is near 2^11 there), 2^-126 in bf16.  Head and remainder differ from p by at most 2^-16 of it (bf16: the remainder
// is below 2^-7, rounded to 8 bits).
template <typename T> __device__ __forceinline__ void split(float p, float q, uint32_t& head, uint32_t& rest);
template <> __device__ __forceinline__ void split<__nv_bfloat16>(float p, float q, uint32_t& head, uint32_t& rest) {
    const uint32_t a = __float_as_uint(p), b = __float_as_uint(q);
    head = __byte_perm(a, b, 0x7632);
    const float x = p - __uint_as_float(a & 0xffff0000u), y = q - __uint_as_float(b & 0xffff0000u);
    rest = umma::pack_bf16(p > 0.f ? fmaxf(x, FLT_MIN) : x, q > 0.f ? fmaxf(y, FLT_MIN) : y);
}
template <> __device__ __forceinline__ void split<__half>(float p, float q, uint32_t& head, uint32_t& rest) {
    constexpr float step = 5.9604644775390625e-8f;      // 2^-24
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(head) : "f"(q), "f"(p));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&head));
    const float x = p - h.x, y = q - h.y;
    const __half2 r = __floats2half2_rn(p >= step ? fmaxf(x, step) : x, q >= step ? fmaxf(y, step) : y);
    rest = *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Where the 16 rows of a tile lie.  IN_PAGE (page size a multiple of 16, or no table): one page and slot.  Else: lane r holds
// those of row r.  Looked up a batch of tiles at a time, and the batch after it already, so that no tile waits for the table.
template <bool IN_PAGE, int KT> struct Pages {
    static constexpr int kBatch = IN_PAGE ? 32 / KT : 2 / KT;      // units per batch
    int id, slot, next_id, next_slot;                    // of this lane's tile or row
    __device__ void fetch(const AttnArgs& a, const Piece& p, int c, int warp, int& page, int& at) const {
        const int lane = threadIdx.x & 31;
        const int tile = IN_PAGE ? lane : lane >> 4;     // of the batch's, KT to a unit
        const int unit = c + tile / KT;
        const int64_t pos = (int64_t)p.base + (((int64_t)unit * kWarps + warp) * KT + tile % KT) * kTile + (IN_PAGE ? 0 : lane & 15);
        page = -1;
        at = 0;
        if (unit < p.c1 && pos < p.n && (IN_PAGE || pos >= p.lo)) {
            if (!a.table) {
                page = p.b; at = (int)pos;
                return;
            }
            const int i = (int)((uint32_t)pos / (uint32_t)a.page_size);
            at = (int)pos - i * a.page_size;
            page = a.table[p.b * a.ts + i];
            if (page < 0 || page >= a.num_pages) {
                atomicCAS(&g_device_status, 0, kStatusBadPage);
                page = -1;
            }
        }
    }
};

template <bool IN_PAGE> struct Tile {
    uint32_t mask;                        // which of its 16 keys count
    int64_t ko, vo;                       // IN_PAGE: offset of row 0
    int64_t krow[2], vrow[4];             // else: offsets of the lane's rows
};

// As many as the registers allow without spilling in the loop (heads of 128: three 1288 us, two 1450 at 64 x 8192-8704 keys;
// of 64 in fp16, ragged: four 237, three 241, five 406).
constexpr int decode_blocks_per_sm(int DP, int NT) { return DP == 64 ? (NT == 1 ? 4 : 3) : DP == 128 ? (NT == 1 ? 3 : 2) : 2; }

template <typename T, int DP, int NT, bool IN_PAGE>
__global__ void __launch_bounds__(kThreads, decode_blocks_per_sm(DP, NT)) decode_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int HP = 8 * NT, KC = DP / 32, VC = DP / 64, MT = DP / 16, PITCH = DP + 4, KT = tiles(DP);
    __shared__ __align__(16) float s_o[kWarps * HP * PITCH];
    __shared__ float s_m[kWarps][HP], s_l[kWarps][HP];
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) a.open[blockIdx.x].b = -1;
    Run run(a);
    const T* kp = static_cast<const T*>(a.k);
    const T* vp = static_cast<const T*>(a.v);
    const bool full_d = a.D == DP;
    while (run.at < run.end) {
        const Piece p = next_piece<HP>(a, run);
        uint4 qf[KC][NT];
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int h = nt * 8 + g, d = i * 32 + t * 8;
                qf[i][nt] = make_uint4(0, 0, 0, 0);
                if (h < p.heads && d < a.D)
                    qf[i][nt] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + p.b * a.qsb + (p.h0 + h) * a.qsh + d);
            }
        float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -FLT_MAX;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
        }
        const T* kh = kp + p.kvh * a.ksh + t * 8;
        const T* vh = vp + p.kvh * a.vsh + g * 8;
        uint4 kr[KT][KC][2], vr[KT][VC][4];
        Pages<IN_PAGE, KT> pages;
        pages.fetch(a, p, p.c0, warp, pages.id, pages.slot);
        pages.fetch(a, p, p.c0 + pages.kBatch, warp, pages.next_id, pages.next_slot);
        int left = pages.kBatch;

        // the warp's tiles of unit c; moves the lookups on
        auto locate = [&](int c, Tile<IN_PAGE> (&tl)[KT]) {
            if (left == 0) {
                pages.id = pages.next_id; pages.slot = pages.next_slot;
                pages.fetch(a, p, c + pages.kBatch, warp, pages.next_id, pages.next_slot);
                left = pages.kBatch;
            }
            const int j = (pages.kBatch - left--) * KT;
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                if (IN_PAGE) {
                    const int64_t pos = (int64_t)p.base + (((int64_t)c * kWarps + warp) * KT + x) * kTile;
                    const int id = __shfl_sync(0xffffffffu, pages.id, j + x), slot = __shfl_sync(0xffffffffu, pages.slot, j + x);
                    tl[x].mask = 0;
                    if (id >= 0) {
                        const int64_t from = p.lo - pos, to = p.n - pos;          // rows from .. to - 1
                        tl[x].mask = to >= 16 ? 0xffffu : (1u << to) - 1u;         // (to > 0 where there is a page)
                        if (from > 0) tl[x].mask &= from >= 16 ? 0u : 0xffffu << from;
                    }
                    tl[x].ko = (int64_t)id * a.ksp + (int64_t)slot * a.kss;
                    tl[x].vo = (int64_t)id * a.vsp + (int64_t)slot * a.vss;
                } else {
                    const int at = (j + x) * 16;
                    tl[x].mask = (__ballot_sync(0xffffffffu, pages.id >= 0) >> at) & 0xffffu;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = at + g + 8 * i;
                        tl[x].krow[i] = (int64_t)__shfl_sync(0xffffffffu, pages.id, r) * a.ksp + (int64_t)__shfl_sync(0xffffffffu, pages.slot, r) * a.kss;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = at + 2 * t + (i & 1) + 8 * (i >> 1);
                        tl[x].vrow[i] = (int64_t)__shfl_sync(0xffffffffu, pages.id, r) * a.vsp + (int64_t)__shfl_sync(0xffffffffu, pages.slot, r) * a.vss;
                    }
                }
            }
        };
        // Rows that do not count are not read, and enter as zeros: whatever lies there stays out.
        auto load_k = [&](const Tile<IN_PAGE> (&tl)[KT]) {
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const T* row = kh + (IN_PAGE ? tl[x].ko + (g + 8 * r) * a.kss : tl[x].krow[r]);
                    if (tl[x].mask == 0xffffu && full_d) {
#pragma unroll
                        for (int i = 0; i < KC; ++i) kr[x][i][r] = ld16(row + i * 32);
                    } else {
                        const bool ok = (tl[x].mask >> (g + 8 * r)) & 1;
#pragma unroll
                        for (int i = 0; i < KC; ++i) {
                            kr[x][i][r] = make_uint4(0, 0, 0, 0);
                            if (ok && i * 32 + t * 8 < a.D) kr[x][i][r] = ld16(row + i * 32);
                        }
                    }
                }
        };
        auto load_v = [&](const Tile<IN_PAGE> (&tl)[KT]) {
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = 2 * t + (r & 1) + 8 * (r >> 1);
                    const T* row = vh + (IN_PAGE ? tl[x].vo + key * a.vss : tl[x].vrow[r]);
                    if (tl[x].mask == 0xffffu && full_d) {
#pragma unroll
                        for (int i = 0; i < VC; ++i) vr[x][i][r] = ld16(row + i * 64);
                    } else {
                        const bool ok = (tl[x].mask >> key) & 1;
#pragma unroll
                        for (int i = 0; i < VC; ++i) {
                            vr[x][i][r] = make_uint4(0, 0, 0, 0);
                            if (ok && i * 64 + g * 8 < a.D) vr[x][i][r] = ld16(row + i * 64);
                        }
                    }
                }
        };

        Tile<IN_PAGE> cur[KT];
        locate(p.c0, cur);
        load_k(cur);
        load_v(cur);
        for (int c = p.c0; c < p.c1; ++c) {
            float s[KT][NT][4];
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[x][nt][0] = s[x][nt][1] = s[x][nt][2] = s[x][nt][3] = 0.f;
#pragma unroll
                    for (int i = 0; i < KC; ++i) {
                        mma<T>(s[x][nt], kr[x][i][0].x, kr[x][i][1].x, kr[x][i][0].y, kr[x][i][1].y, qf[i][nt].x, qf[i][nt].y);
                        mma<T>(s[x][nt], kr[x][i][0].z, kr[x][i][1].z, kr[x][i][0].w, kr[x][i][1].w, qf[i][nt].z, qf[i][nt].w);
                    }
                }
            Tile<IN_PAGE> nxt[KT];
            const bool more = c + 1 < p.c1;
            if (more) {
                locate(c + 1, nxt);
                load_k(nxt);
            }
            bool up = false;
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[x][nt][i] *= a.scale;
                    if (cur[x].mask != 0xffffu) {
                        if (!((cur[x].mask >> g) & 1)) s[x][nt][0] = s[x][nt][1] = -INFINITY;
                        if (!((cur[x].mask >> (g + 8)) & 1)) s[x][nt][2] = s[x][nt][3] = -INFINITY;
                    }
                    constexpr float over = Ref<T>::shift + Ref<T>::slack;
                    up |= fmaxf(s[x][nt][0], s[x][nt][2]) > m[nt][0] + over || fmaxf(s[x][nt][1], s[x][nt][3]) > m[nt][1] + over;
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float z = fmaxf(s[0][nt][i], s[0][nt][i + 2]);
#pragma unroll
                        for (int x = 1; x < KT; ++x) z = fmaxf(z, fmaxf(s[x][nt][i], s[x][nt][i + 2]));
                        z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, 4));
                        z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, 8));
                        z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, 16));
                        z = fmaxf(z - Ref<T>::shift, m[nt][i]);
                        const float f = exp2f(m[nt][i] - z);
                        m[nt][i] = z;
                        l[nt][i] *= f;
#pragma unroll
                        for (int j = 0; j < MT; ++j) { o[j][nt][i] *= f; o[j][nt][i + 2] *= f; }
                    }
            }
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float p0 = exp2f(s[x][nt][2 * i] - m[nt][0]), p1 = exp2f(s[x][nt][2 * i + 1] - m[nt][1]);
                        l[nt][0] += p0;
                        l[nt][1] += p1;
                        uint32_t head, rest;
                        split<T>(p0, p1, head, rest);
                        ph[nt][i] = transpose8(head);
                        pl[nt][i] = transpose8(rest);
                    }
#pragma unroll
                for (int i = 0; i < VC; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t r0 = word(vr[x][i][0], j), r1 = word(vr[x][i][1], j), r2 = word(vr[x][i][2], j), r3 = word(vr[x][i][3], j);
                        const uint32_t a0 = __byte_perm(r0, r1, 0x5410), a1 = __byte_perm(r0, r1, 0x7632);
                        const uint32_t a2 = __byte_perm(r2, r3, 0x5410), a3 = __byte_perm(r2, r3, 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma<T>(o[i * 4 + j][nt], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                            mma<T>(o[i * 4 + j][nt], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                        }
                    }
            }
            if (more) {
                load_v(nxt);
#pragma unroll
                for (int x = 0; x < KT; ++x) cur[x] = nxt[x];
            }
        }

        __syncthreads();                                            // (the previous piece's sums have been read)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = l[nt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int h = nt * 8 + 2 * t + i;
                if (g == 0) { s_m[warp][h] = m[nt][i]; s_l[warp][h] = x; }
                float* row = s_o + (warp * HP + h) * PITCH + g * 8;
#pragma unroll
                for (int v = 0; v < VC; ++v) {
                    *reinterpret_cast<float4*>(row + v * 64) = make_float4(o[v * 4][nt][i], o[v * 4][nt][i + 2], o[v * 4 + 1][nt][i], o[v * 4 + 1][nt][i + 2]);
                    *reinterpret_cast<float4*>(row + v * 64 + 4) = make_float4(o[v * 4 + 2][nt][i], o[v * 4 + 2][nt][i + 2], o[v * 4 + 3][nt][i], o[v * 4 + 3][nt][i + 2]);
                }
            }
        __syncthreads();
        join_warps<T, DP, HP, PITCH>(a, p, run, s_o, s_m, s_l, true);
    }
}

// ---- any type, head size and alignment: fp32 products on the CUDA cores ----------------------------------------------------
// Eight lanes hold a key, a lane the values 32 i + 4 (lane % 8) .. + 3 of it; a warp works on four keys at a time, each group
// of eight lanes with a maximum and sums of its own.  Up to four query heads at a time; one alone leaves registers for more
// keys in flight.  fp32, 16 sequences of 4000-8000 keys, 16 heads of 128: 229 us (1.0); 32 sequences, 16 to 32 over 8 heads:
// 359-376 us (0.65: issue slots, and one step in flight), 40 to 64 over 8: 676-699 us (0.36: two passes); heads of 64, 32 and 64
// over 8: 208 and 406 us (0.55, 0.30); of 256, 16 and 32 over 4: 393 and 717 us (0.60, 0.32).  bf16 heads of 44, 16 over 16: 374
// us (0.22: no 16-byte vectors of eight values, so not the tensor cores).
template <typename T, bool VEC> __device__ __forceinline__ float4 load4(const T* p, int d, int D) {
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) {
        if (d < D) {
            if (sizeof(T) == 4) return *reinterpret_cast<const float4*>(p + d);
            const uint2 u = *reinterpret_cast<const uint2*>(p + d);
            const T* t = reinterpret_cast<const T*>(&u);
            r = make_float4(to_f32<T>(t[0]), to_f32<T>(t[1]), to_f32<T>(t[2]), to_f32<T>(t[3]));
        }
    } else {
        if (d < D) r.x = to_f32<T>(p[d]);
        if (d + 1 < D) r.y = to_f32<T>(p[d + 1]);
        if (d + 2 < D) r.z = to_f32<T>(p[d + 2]);
        if (d + 3 < D) r.w = to_f32<T>(p[d + 3]);
    }
    return r;
}

constexpr int any_blocks_per_sm(int DP, int HP) { return DP == 256 ? (HP == 1 ? 3 : 2) : 4; }

// Scratch: (sums, m, l) of two open pieces a block, and what is open.
constexpr int64_t scratch_bytes(int64_t blocks, int DP, int HP) { return blocks * 2 * HP * (DP * 4 + 8) + blocks * (int64_t)sizeof(Open); }
constexpr bool scratch_fits() {
    for (int DP = 64; DP <= 256; DP *= 2) {
        for (int NT = 1; NT <= 2; ++NT)
            if (scratch_bytes(kNumSMs * decode_blocks_per_sm(DP, NT), DP, 8 * NT) > VTX_PAGED_DECODE_SCRATCH_MAX && !(DP == 256 && NT == 2)) return false;
        for (int HP = 1; HP <= 4; HP += 3)
            if (scratch_bytes(kNumSMs * any_blocks_per_sm(DP, HP), DP, HP) > VTX_PAGED_DECODE_SCRATCH_MAX) return false;
    }
    return true;
}
static_assert(scratch_fits(), "VTX_PAGED_DECODE_SCRATCH_MAX");

template <typename T, int DP, int HP, bool VEC>
__global__ void __launch_bounds__(kThreads, any_blocks_per_sm(DP, HP)) decode_any_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int C = DP / 32, PITCH = DP + 4, STEPS = HP == 1 ? 256 / DP : DP == 64 ? 2 : 1;
    __shared__ __align__(16) float s_o[kWarps * HP * PITCH], s_q[HP * DP];
    __shared__ float s_m[kWarps][HP], s_l[kWarps][HP];
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & 7, kq = lane >> 3;
    if (threadIdx.x == 0) a.open[blockIdx.x].b = -1;
    Run run(a);
    while (run.at < run.end) {
        const Piece p = next_piece<HP>(a, run);
        __syncthreads();
        for (int i = threadIdx.x; i < HP * DP; i += kThreads) {
            const int h = i / DP, d = i - h * DP;
            s_q[i] = h < p.heads && d < a.D ? to_f32<T>(static_cast<const T*>(a.q)[p.b * a.qsb + (p.h0 + h) * a.qsh + d]) : 0.f;
        }
        __syncthreads();
        float m[HP], l[HP];
        float4 o[HP][C];
#pragma unroll
        for (int h = 0; h < HP; ++h) {
            m[h] = -FLT_MAX;
            l[h] = 0.f;
#pragma unroll
            for (int i = 0; i < C; ++i) o[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const T* kh = static_cast<const T*>(a.k) + p.kvh * a.ksh;
        const T* vh = static_cast<const T*>(a.v) + p.kvh * a.vsh;
        for (int c = p.c0; c < p.c1; ++c) {
            for (int step = 0; step < kTile / 4; step += STEPS) {
                float4 kv[STEPS][C], vv[STEPS][C];
                bool ok[STEPS];
#pragma unroll
                for (int u = 0; u < STEPS; ++u) {
                    const int64_t pos = (int64_t)p.base + ((int64_t)c * kWarps + warp) * kTile + (step + u) * 4 + kq;
                    int page = p.b, at = (int)pos;
                    ok[u] = pos >= p.lo && pos < p.n;
                    if (ok[u] && a.table) {
                        const int i = (int)((uint32_t)pos / (uint32_t)a.page_size);
                        at = (int)pos - i * a.page_size;
                        page = a.table[p.b * a.ts + i];
                        if (page < 0 || page >= a.num_pages) {
                            atomicCAS(&g_device_status, 0, kStatusBadPage);
                            ok[u] = false;
                        }
                    }
                    const T* kk = kh + page * a.ksp + at * a.kss;
                    const T* vk = vh + page * a.vsp + at * a.vss;
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        kv[u][i] = vv[u][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (ok[u]) {
                            kv[u][i] = load4<T, VEC>(kk, i * 32 + sub * 4, a.D);
                            vv[u][i] = load4<T, VEC>(vk, i * 32 + sub * 4, a.D);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < STEPS; ++u)
#pragma unroll
                    for (int h = 0; h < HP; ++h) {
                        float s = 0.f;
#pragma unroll
                        for (int i = 0; i < C; ++i) {
                            const float4 q = *reinterpret_cast<const float4*>(s_q + h * DP + i * 32 + sub * 4);
                            s += q.x * kv[u][i].x + q.y * kv[u][i].y + q.z * kv[u][i].z + q.w * kv[u][i].w;
                        }
                        s += __shfl_xor_sync(0xffffffffu, s, 1);
                        s += __shfl_xor_sync(0xffffffffu, s, 2);
                        s += __shfl_xor_sync(0xffffffffu, s, 4);
                        s = ok[u] ? s * a.scale : -INFINITY;
                        if (s > m[h] + Ref<float>::shift + Ref<float>::slack) {
                            const float f = exp2f(m[h] - s);
                            m[h] = s;
                            l[h] *= f;
#pragma unroll
                            for (int i = 0; i < C; ++i) { o[h][i].x *= f; o[h][i].y *= f; o[h][i].z *= f; o[h][i].w *= f; }
                        }
                        const float e = exp2f(s - m[h]);
                        l[h] += e;
#pragma unroll
                        for (int i = 0; i < C; ++i) {
                            o[h][i].x += e * vv[u][i].x; o[h][i].y += e * vv[u][i].y;
                            o[h][i].z += e * vv[u][i].z; o[h][i].w += e * vv[u][i].w;
                        }
                    }
            }
        }
        // the four groups of a warp, then the warps
#pragma unroll
        for (int h = 0; h < HP; ++h) {
            float x = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float f = exp2f(m[h] - x);
            auto sum = [&](float v) {
                v *= f;
                v += __shfl_xor_sync(0xffffffffu, v, 8);
                return v + __shfl_xor_sync(0xffffffffu, v, 16);
            };
            const float lt = sum(l[h]);
            if (lane == 0) { s_m[warp][h] = x; s_l[warp][h] = lt; }
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const float4 r = make_float4(sum(o[h][i].x), sum(o[h][i].y), sum(o[h][i].z), sum(o[h][i].w));
                if (kq == 0) *reinterpret_cast<float4*>(s_o + (warp * HP + h) * PITCH + i * 32 + sub * 4) = r;
            }
        }
        __syncthreads();
        join_warps<T, DP, HP, PITCH>(a, p, run, s_o, s_m, s_l, false);
    }
}

// ---- the open (sequence, head group)s: block (w, h) joins head h of the one that begins in run w ----------------------------
template <typename T, int DP, int HP> __global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ AttnArgs a, int W) {
    constexpr int Q = DP / 4, R = kThreads / Q;                      // threads to a row of sums; rows at a time
    __shared__ float2 s_ml[R];
    __shared__ __align__(16) float s_o[R][DP];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int w0 = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, q = tid % Q, r0 = tid / Q;
    const int run0 = w0 / a.abreast, runs = W / a.abreast;
    // the run it begins in keeps it in slot 1, the others in slot 0
    auto row = [&](int i) { return ((int64_t)(w0 + i * a.abreast) * 2 + (i == 0)) * HP + h; };
    // the first rows are loaded before it is known whether this block has any (9.8 -> 8.7 us at one sequence of 700 keys)
    constexpr int AHEAD = 4;
    float2 ml[AHEAD];
    float4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (run0 + r0 + j * R < runs) {
            ml[j] = a.part_ml[row(r0 + j * R)];
            x[j] = *reinterpret_cast<const float4*>(a.part + row(r0 + j * R) * DP + q * 4);
        }
    const Open op = a.open[w0];
    if (op.b < 0) return;
    const int kvh = op.hg / a.passes, first = (op.hg - kvh * a.passes) * HP;
    if (first + h >= a.G) return;
    const int n = op.runs;
    // a run may be empty where there are fewer units than runs
    const bool sparse = op.units < runs;
    auto empty = [&](int i) { return run_start(op.units, run0 + i, runs) == run_start(op.units, run0 + i + 1, runs); };
    float m = -FLT_MAX, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float2& ml, const float4& x) {
        const float top = fmaxf(m, ml.x), f = exp2f(m - top), g = exp2f(ml.x - top);
        o.x = o.x * f + x.x * g; o.y = o.y * f + x.y * g; o.z = o.z * f + x.z * g; o.w = o.w * f + x.w * g;
        l = l * f + ml.y * g;
        m = top;
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (r0 + j * R < n && !(sparse && empty(r0 + j * R))) add(ml[j], x[j]);
#pragma unroll 4
    for (int i = r0 + AHEAD * R; i < n; i += R)
        if (!(sparse && empty(i))) add(a.part_ml[row(i)], *reinterpret_cast<const float4*>(a.part + row(i) * DP + q * 4));
    if (q == 0) s_ml[r0] = make_float2(m, l);
    *reinterpret_cast<float4*>(&s_o[r0][q * 4]) = o;
    __syncthreads();
    m = -FLT_MAX;
    for (int i = 0; i < R; ++i) m = fmaxf(m, s_ml[i].x);
    l = 0.f;
    for (int i = 0; i < R; ++i) l += s_ml[i].y * exp2f(s_ml[i].x - m);
    const int head = kvh * a.G + first + h;
    float none = 0.f;
    if (l == 0.f) {
        const Seq s(a, op.b);
        none = zero_sum(a, op.b, s.lo, s.n);
    }
    T* y = static_cast<T*>(a.out) + op.b * a.osb + head * a.osh;
    for (int d = tid; d < a.D; d += kThreads) {
        float x = 0.f;
        for (int i = 0; i < R; ++i) x += s_o[i][d] * exp2f(s_ml[i].x - m);
        y[d] = from_f32<T>(l == 0.f ? none : x / l);
    }
    if (tid == 0 && a.lse) a.lse[(int64_t)op.b * a.Hq + head] = (m + log2f(l)) * 0.69314718055994531f;
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Plan {
    int DP, HP, blocks, unit, abreast;
    bool tensor, in_page, vec;
    int64_t slots, bytes;
};

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int64_t es, int64_t n) {
    return reinterpret_cast<uintptr_t>(p) % n == 0 && (a * es) % n == 0 && (b * es) % n == 0 && (c * es) % n == 0;
}

Plan make_plan(const vtx_paged_decode_params& p) {
    Plan pl{};
    const int64_t es = dtype_size(p.io_dtype), G = p.Hq / p.Hk;
    pl.DP = p.D <= 64 ? 64 : p.D <= 128 ? 128 : 256;
    pl.tensor = es == 2 && p.D % 8 == 0 && aligned(p.q, p.q_stride_b, p.q_stride_h, 0, es, 16) &&
                aligned(p.k_pages, p.k_stride_page, p.k_stride_slot, p.k_stride_head, es, 16) &&
                aligned(p.v_pages, p.v_stride_page, p.v_stride_slot, p.v_stride_head, es, 16) &&
                aligned(p.out, p.out_stride_b, p.out_stride_h, 0, es, 8);
    pl.in_page = !p.block_table || p.page_size % kTile == 0;
    pl.vec = p.D % 4 == 0 && aligned(p.k_pages, p.k_stride_page, p.k_stride_slot, p.k_stride_head, es, 4 * es) &&
             aligned(p.v_pages, p.v_stride_page, p.v_stride_slot, p.v_stride_head, es, 4 * es);
    int per_sm;
    if (pl.tensor) {
        // 9 to 16 query heads of a key head share a pass (but for heads of 256 values, whose sums fill the registers)
        const int NT = G > 8 && pl.DP < 256 ? 2 : 1;
        pl.HP = 8 * NT;
        per_sm = decode_blocks_per_sm(pl.DP, NT);
    } else {
        pl.HP = G > 1 ? 4 : 1;
        per_sm = any_blocks_per_sm(pl.DP, pl.HP);
    }
    // no more blocks than units
    const int64_t keys = p.block_table ? p.table_width * p.page_size : p.page_size;
    pl.unit = unit_keys(pl.DP, pl.tensor);
    const int64_t per_seq = ceil_div<int64_t>(keys < INT32_MAX ? keys : INT32_MAX, pl.unit) + 1;
    const int64_t pairs = p.B * p.Hk * ceil_div<int64_t>(G, pl.HP);
    int64_t most = pairs > (1 << 20) ? pairs : pairs * (per_seq > 0 ? per_seq : 1);
    pl.blocks = (int)(most < (int64_t)kNumSMs * per_sm ? most : (int64_t)kNumSMs * per_sm);
    const int64_t groups = p.Hk * ceil_div<int64_t>(G, pl.HP);
    // Head groups abreast -- the blocks of a run walk the same keys of all heads side by side, whose rows are neighbours in
    // memory -- where that leaves no more than a twentieth of the blocks out, or where rows share 128-byte lines, which DRAM
    // delivers whole.  Else all heads' units in one row.  (us abreast / in a row: 1,048,576 keys x 8 heads 631 / 651, ragged 8
    // heads of 64 224 / 248, 256 sequences of 100-600 keys 76 / 81, 16 heads of 112 262 / 297, of 80 234 / 252; 64 x 8192-8704
    // keys x 32 heads, 416 of 444 blocks, 1325 / 1306.)
    const bool lines = (p.D * es) % 128 == 0;
    pl.abreast = groups <= pl.blocks && (pl.blocks % groups * 20 <= pl.blocks || !lines) ? (int)groups : 1;
    pl.blocks -= pl.blocks % pl.abreast;
    pl.slots = (int64_t)pl.blocks * 2 * pl.HP;
    pl.bytes = scratch_bytes(pl.blocks, pl.DP, pl.HP);
    return pl;
}

template <typename T, int DP, int HP> int launch_join(const AttnArgs& a, int W, cudaStream_t s) {
    if (int rc = check_launch("paged_decode_attention")) return rc;          // (nothing was written that could be joined)
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)W, (unsigned)(a.G < HP ? a.G : HP));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, join_kernel<T, DP, HP>, a, W);
    return check_launch("paged_decode_attention");
}

template <typename T, int DP> int launch_tensor(const AttnArgs& a, const Plan& pl, cudaStream_t s) {
    const unsigned W = (unsigned)pl.blocks;
    if (pl.HP == 8) {
        if (pl.in_page) decode_kernel<T, DP, 1, true><<<W, kThreads, 0, s>>>(a);
        else decode_kernel<T, DP, 1, false><<<W, kThreads, 0, s>>>(a);
        return launch_join<T, DP, 8>(a, (int)W, s);
    }
    if constexpr (DP < 256) {
        if (pl.in_page) decode_kernel<T, DP, 2, true><<<W, kThreads, 0, s>>>(a);
        else decode_kernel<T, DP, 2, false><<<W, kThreads, 0, s>>>(a);
        return launch_join<T, DP, 16>(a, (int)W, s);
    }
    return fail(VTX_ERR_UNSUPPORTED, "paged_decode_attention: no kernel");
}

template <typename T, int DP> int launch_any(const AttnArgs& a, const Plan& pl, cudaStream_t s) {
    const unsigned W = (unsigned)pl.blocks;
    if (pl.HP == 1) {
        if (pl.vec) decode_any_kernel<T, DP, 1, true><<<W, kThreads, 0, s>>>(a);
        else decode_any_kernel<T, DP, 1, false><<<W, kThreads, 0, s>>>(a);
        return launch_join<T, DP, 1>(a, (int)W, s);
    }
    if (pl.vec) decode_any_kernel<T, DP, 4, true><<<W, kThreads, 0, s>>>(a);
    else decode_any_kernel<T, DP, 4, false><<<W, kThreads, 0, s>>>(a);
    return launch_join<T, DP, 4>(a, (int)W, s);
}

int validate(const vtx_paged_decode_params* p) {
    VTX_REQUIRE(p, VTX_ERR_BAD_ARG, "paged_decode_attention: null pointer");
    VTX_REQUIRE(valid_dtype(p->io_dtype), VTX_ERR_BAD_ARG, "paged_decode_attention: unknown io dtype %lld", (long long)p->io_dtype);
    VTX_REQUIRE(p->B >= 0 && p->Hk > 0 && p->Hq > 0 && p->D > 0 && p->page_size > 0 && p->num_pages >= 0 && p->table_width >= 0,
                VTX_ERR_BAD_ARG, "paged_decode_attention: bad sizes");
    VTX_REQUIRE(p->Hq % p->Hk == 0, VTX_ERR_BAD_ARG, "paged_decode_attention: %lld query heads for %lld key heads",
                (long long)p->Hq, (long long)p->Hk);
    VTX_REQUIRE(p->D <= 256, VTX_ERR_UNSUPPORTED, "paged_decode_attention: heads of %lld > 256 values", (long long)p->D);
    VTX_REQUIRE(p->window >= 0, VTX_ERR_BAD_ARG, "paged_decode_attention: negative window");
    VTX_REQUIRE(p->B < (1 << 24) && p->Hq < (1 << 16) && p->num_pages < INT32_MAX && p->page_size < INT32_MAX, VTX_ERR_UNSUPPORTED,
                "paged_decode_attention: more than 2^24 sequences, 2^16 heads or 2^31 pages or slots");
    VTX_REQUIRE(p->block_table || p->num_pages >= p->B, VTX_ERR_BAD_ARG, "paged_decode_attention: %lld sequences, %lld pages and no block table",
                (long long)p->B, (long long)p->num_pages);
    return VTX_OK;
}

}  // namespace
}  // namespace vtx

extern "C" int64_t vtx_paged_decode_scratch_bytes(const vtx_paged_decode_params* p) {
    if (vtx::validate(p) != VTX_OK) return 0;
    return p->B ? vtx::make_plan(*p).bytes : 0;
}

extern "C" int vtx_paged_decode_attention(const vtx_paged_decode_params* p, void* stream) {
    using namespace vtx;
    if (int rc = validate(p)) return rc;
    if (p->B == 0) return VTX_OK;
    VTX_REQUIRE(p->q && p->out && p->seqlens && (p->num_pages == 0 || (p->k_pages && p->v_pages)), VTX_ERR_BAD_ARG,
                "paged_decode_attention: null pointer");
    VTX_REQUIRE(p->scratch && reinterpret_cast<uintptr_t>(p->scratch) % 16 == 0, VTX_ERR_BAD_ARG,
                "paged_decode_attention: scratch needed (vtx_paged_decode_scratch_bytes, 16-byte aligned)");
    const Plan pl = make_plan(*p);
    AttnArgs a{};
    a.q = p->q; a.qsb = p->q_stride_b; a.qsh = p->q_stride_h;
    a.k = p->k_pages; a.ksp = p->k_stride_page; a.kss = p->k_stride_slot; a.ksh = p->k_stride_head;
    a.v = p->v_pages; a.vsp = p->v_stride_page; a.vss = p->v_stride_slot; a.vsh = p->v_stride_head;
    a.table = p->block_table; a.ts = p->table_stride; a.lens = p->seqlens;
    a.out = p->out; a.osb = p->out_stride_b; a.osh = p->out_stride_h; a.lse = p->lse;
    char* w = static_cast<char*>(p->scratch);
    a.part = reinterpret_cast<float*>(w);
    a.part_ml = reinterpret_cast<float2*>(w + pl.slots * pl.DP * 4);
    a.open = reinterpret_cast<Open*>(w + pl.slots * (pl.DP * 4 + 8));
    a.scale = (float)(p->softmax_scale * 1.44269504088896340736);
    a.window = p->window > 0 && p->window < INT32_MAX ? (int)p->window : INT32_MAX;
    a.B = (int)p->B; a.Hq = (int)p->Hq; a.G = (int)(p->Hq / p->Hk); a.D = (int)p->D;
    a.page_size = (int)p->page_size; a.num_pages = (int)p->num_pages;
    a.passes = (a.G + pl.HP - 1) / pl.HP;
    a.unit = pl.unit;
    a.abreast = pl.abreast;
    a.head_groups = (int)p->Hk * a.passes;
    a.max_keys = p->block_table ? p->table_width * p->page_size : p->page_size;
    cudaStream_t s = (cudaStream_t)stream;
    if (pl.tensor) {
        if (p->io_dtype == VTX_BF16)
            return pl.DP == 64 ? launch_tensor<__nv_bfloat16, 64>(a, pl, s) : pl.DP == 128 ? launch_tensor<__nv_bfloat16, 128>(a, pl, s)
                                                                              : launch_tensor<__nv_bfloat16, 256>(a, pl, s);
        return pl.DP == 64 ? launch_tensor<__half, 64>(a, pl, s) : pl.DP == 128 ? launch_tensor<__half, 128>(a, pl, s) : launch_tensor<__half, 256>(a, pl, s);
    }
    VTX_DISPATCH_IO(p->io_dtype, T, {
        return pl.DP == 64 ? launch_any<T, 64>(a, pl, s) : pl.DP == 128 ? launch_any<T, 128>(a, pl, s) : launch_any<T, 256>(a, pl, s);
    });
    return VTX_OK;
}
