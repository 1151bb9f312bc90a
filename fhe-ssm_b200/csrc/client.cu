// client.cu -- the client's token step on the GPU: the head product with a 4-bit table, the choice of
// the next token, and the look-up of the next embedding row in the same (tied) table.
//
// The server returns encrypted normed rows; the client decrypts them, applies the tied head in plaintext
// (the --dec-out side of gpu_real_model.cu:2444-2533), picks a token (spec_decode/decode_policy.py:37) and
// embeds it with a row of the same table (ml-eval/fhe_client.py:123-135).
//
// All three run on a stream of the caller's choice, allocate nothing and read nothing of the context's
// chain or keys.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace fhe {

// one value of a tensor whose type is known at run time (FHE_F32, FHE_F16, FHE_BF16)
__device__ __forceinline__ float ld_any(const void* p, int type, long long i) {
    if (type == FHE_F32) return static_cast<const float*>(p)[i];
    if (type == FHE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void st_any(void* p, int type, long long i, float v) {
    if (type == FHE_F32) static_cast<float*>(p)[i] = v;
    else if (type == FHE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Lets kernel K have all the shared memory a block can; asked of the driver once per GPU.
template <auto K>
static void client_smem(const Context& cx) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << cx.device;
    if (done.load(std::memory_order_relaxed) & bit) return;
    CUDA_CHECK(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
    done.fetch_or(bit, std::memory_order_relaxed);
}

// ---- products with a 4-bit table -----------------------------------------------------------
// W[i][c] = s[i][c / group] (q[i][c] - 8); out[r][i] = sum_c x[r][c] W[i][c].
//
// Within a group the sum is a product of whole numbers -8..7, which every 16-bit float holds exactly, with x; the
// scale is applied to the group's sum in float32.  x is cut into bf16 pieces that add up to it exactly (float32: 3 of 8
// bits, float16: 2, bf16: itself), each piece a column of the matrix product, so nothing is rounded before the
// float32 sums.
//
// k_q4_mma: few columns (one row of x, or some).  What it must read is the table, so a warp streams 16 table rows through a
// shared-memory ring of its own (cp.async, no block barrier) and multiplies them on the tensor cores (m16n8k16: 16 table
// rows x 8 columns of pieces); with a CUDA-core product the unpacking and the float32 multiply-adds, 4 instructions
// a value, would cost more than the table's bytes.  Columns are permuted so that a 32-bit word of
// 8 values is a lane's share of two steps: the pairs (0,4), (1,5), (2,6), (3,7) come out of the word by one
// mask each.  Several warps share 16 rows where the table is short, each a part of the columns.
constexpr int kQ4Warps = 8, kQ4Threads = 32 * kQ4Warps;
constexpr int kQ4Stage = 4;             // 32-column chunks of a stage
constexpr int kQ4Stages = 4;
constexpr int kQ4Pitch = kQ4Stage * 16 + 16;   // bytes of a row in a stage: 20 banks apart, 8 rows x 4 words meet all 32
constexpr int kQ4StageBytes = 16 * kQ4Pitch;
constexpr int kQ4RingBytes = kQ4Warps * kQ4Stages * kQ4StageBytes;
constexpr int kQ4MaxBytes = 163840;     // shared memory for x's pieces and the scales

struct Q4Args {
    fhe_q4 w;
    const void* x;
    int xt, terms, m;
    long long ldx;
    void* out;
    int ot;
    long long ldo;
    int per;         // rows of x that a block takes
    int ks_log2;     // 2^ks_log2 warps share a row tile's columns
    int kb_chunks;   // chunks of columns held at a time, in whole stages for each of these warps
    int units;       // scales that a warp holds for each row
    uint32_t group_magic;   // chunk / (chunks of a group) = chunk * magic >> 32 (both at most 2^15); 0: a group is a chunk
    int wide;        // rows of x start on 16-byte boundaries
};

// The first bf16 piece of v (its bits), and what is left of v: pieces are cut, not rounded, so none overflows; an infinity or
// NaN is all in the first.
__device__ __forceinline__ uint32_t q4_piece(float& v) {
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7f800000u) == 0x7f800000u) {
        v = 0.f;
        return b & 0x007fffffu ? 0x7fffu : b >> 16;
    }
    v -= __uint_as_float(b & 0xffff0000u);
    return b >> 16;
}

template <class T>
__device__ __forceinline__ float q4_float(T v);
template <>
__device__ __forceinline__ float q4_float(float v) { return v; }
template <>
__device__ __forceinline__ float q4_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float q4_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Pieces of rows r0..r0+mr of x, chunks kb0..kb1 -> the product's operand [chunk][tile of 8 columns][lane], 16 bytes each:
// the lane's column (r TERMS + piece) and its 8 values, paired as q4_unpack pairs the table's.
template <class T, int TERMS>
__device__ __forceinline__ void q4_cut(const Q4Args& a, uint4* xs, int nt, int r0, int mr, int kb0, int kb1) {
    // a warp takes 8 chunks of a row at a time
    const int lane = threadIdx.x & 31, t = lane & 3;
    int r = threadIdx.x >> 5, ch = lane >> 2;
    for (;; r += kQ4Warps) {
        while (r >= mr) r -= mr, ch += 8;
        if (ch - (lane >> 2) >= kb1 - kb0) break;
        if (ch >= kb1 - kb0) continue;
        const int k = (kb0 + ch) * 32 + t * 8;
        const T* src = static_cast<const T*>(a.x) + (r0 + r) * a.ldx + k;
        float v[8];
        if (a.wide && k + 8 <= a.w.cols) {
            T u[8];
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) * 8 / 16; j++)
                reinterpret_cast<uint4*>(u)[j] = reinterpret_cast<const uint4*>(src)[j];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = q4_float(u[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = k + j < a.w.cols ? q4_float(src[j]) : 0.f;
        }
#pragma unroll
        for (int term = 0; term < TERMS; term++) {
            uint32_t p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) p[j] = q4_piece(v[j]);
            const int col = r * TERMS + term;
            xs[(ch * nt + (col >> 3)) * 32 + (col & 7) * 4 + t] =
                make_uint4(p[0] | p[4] << 16, p[1] | p[5] << 16, p[2] | p[6] << 16, p[3] | p[7] << 16);
        }
    }
}

// 8 values of 4 bits -> bf16 pairs (0,4), (1,5), (2,6), (3,7) of q - 8: 0x4300 is 128, its last bits count in ones
__device__ __forceinline__ void q4_unpack(uint32_t w, uint32_t* p) {
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = (w >> (4 * i) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
        p[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

__device__ __forceinline__ void q4_mma(float* d, const float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Scales of 16 rows (from row0) for `units` units of P chunks from chunk c0 -> sc[unit][row]; 0 past the last column
template <class S, int P>
__device__ __forceinline__ void q4_scales(const fhe_q4& w, uint32_t magic, float* sc, int row0, int c0, int units,
                                          int chunks) {
    const int lane = threadIdx.x & 31;
    const S* src = static_cast<const S*>(w.scale) + (long long)min(row0 + (lane & 15), w.rows - 1) * w.lds;
#pragma unroll 4
    for (int u = lane >> 4; u < units; u += 2) {
        const int ch = c0 + u * P;
        sc[u * 16 + (lane & 15)] = ch < chunks ? q4_float(src[magic ? __umulhi(ch, magic) : ch]) : 0.f;
    }
}

// NT: tiles of 8 columns.  P: chunks after which the scale is applied, the largest of 1, 2, 4 that divides a group's.
template <int NT, int P>
__global__ void __launch_bounds__(kQ4Threads) k_q4_mma(const Q4Args a) {
    extern __shared__ __align__(16) uint8_t qsm[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = qsm + warp * (kQ4Stages * kQ4StageBytes);
    uint4* xs = reinterpret_cast<uint4*>(qsm + kQ4RingBytes);
    const int chunks = (a.w.cols + 31) / 32;
    const int ks = 1 << a.ks_log2, rows = 16 * kQ4Warps >> a.ks_log2;   // warps on a tile, table rows of a block
    const int row0 = blockIdx.x * rows + (warp >> a.ks_log2) * 16, kq = warp & (ks - 1);
    const int r0 = blockIdx.y * a.per, mr = min(a.per, a.m - r0);
    float* sc = reinterpret_cast<float*>(xs + a.kb_chunks * NT * 32) + warp * 16 * a.units;   // [unit][16 rows]
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[n][j] = 0.f;
    // a lane copies 16 bytes of rows g and g + 8 a stage; rows past the end read the last one and are not stored
    const uint8_t* src0 = a.w.q + (long long)min(row0 + g, a.w.rows - 1) * a.w.ldq;
    const uint8_t* src1 = a.w.q + (long long)min(row0 + g + 8, a.w.rows - 1) * a.w.ldq;
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring) + g * kQ4Pitch + t * 16;
    const uint8_t* words = ring + g * kQ4Pitch + t * 4;

    for (int kb0 = 0; kb0 < chunks; kb0 += a.kb_chunks) {
        // the last block may pass the end: values and scales are 0 there
        const int kb1 = kb0 + a.kb_chunks, each = a.kb_chunks >> a.ks_log2, stages = each / kQ4Stage;
        const int c0 = kb0 + kq * each, c1 = c0 + each;
        auto fetch = [&](int s) {
            const int at = c0 + s * kQ4Stage + t;
            if (at < min(c1, chunks)) {
                const uint32_t d = dst + (s % kQ4Stages) * kQ4StageBytes;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src0 + at * 16) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 8 * kQ4Pitch), "l"(src1 + at * 16)
                             : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int s = 0; s < kQ4Stages - 1; s++) fetch(s);
        if (a.w.scale_type == FHE_F16) q4_scales<__half, P>(a.w, a.group_magic, sc, row0, c0, (c1 - c0) / P, chunks);
        else if (a.w.scale_type == FHE_BF16) q4_scales<__nv_bfloat16, P>(a.w, a.group_magic, sc, row0, c0, (c1 - c0) / P, chunks);
        else q4_scales<float, P>(a.w, a.group_magic, sc, row0, c0, (c1 - c0) / P, chunks);
        __syncthreads();   // the previous block's pieces are read
        if (a.xt == FHE_F32) q4_cut<float, 3>(a, xs, NT, r0, mr, kb0, kb1);
        else if (a.xt == FHE_F16) q4_cut<__half, 2>(a, xs, NT, r0, mr, kb0, kb1);
        else q4_cut<__nv_bfloat16, 1>(a, xs, NT, r0, mr, kb0, kb1);
        __syncthreads();
        const uint4* xc = xs + (size_t)(c0 - kb0) * NT * 32 + lane;
        const float* su = sc + g;
        for (int s = 0; s < stages; s++) {
            fetch(s + kQ4Stages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kQ4Stages - 1) : "memory");
            __syncwarp();
            const uint8_t* st = words + (s % kQ4Stages) * kQ4StageBytes;
            constexpr float zero[4] = {0.f, 0.f, 0.f, 0.f};
            float c[NT][4];
#pragma unroll
            for (int ch = 0; ch < kQ4Stage; ch++) {
                uint32_t p[4], q[4];
                q4_unpack(*reinterpret_cast<const uint32_t*>(st + ch * 16), p);
                q4_unpack(*reinterpret_cast<const uint32_t*>(st + 8 * kQ4Pitch + ch * 16), q);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 b = xc[(ch * NT + n) * 32];
                    q4_mma(c[n], ch % P == 0 ? zero : c[n], p[0], q[0], p[1], q[1], b.x, b.y);
                    q4_mma(c[n], c[n], p[2], q[2], p[3], q[3], b.z, b.w);
                }
                if (ch % P == P - 1) {
                    const float sg = su[ch / P * 16], sh = su[ch / P * 16 + 8];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        acc[n][0] += sg * c[n][0];
                        acc[n][1] += sg * c[n][1];
                        acc[n][2] += sh * c[n][2];
                        acc[n][3] += sh * c[n][3];
                    }
                }
            }
            xc += kQ4Stage * NT * 32;
            su += kQ4Stage / P * 16;
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // [warp][column][16 rows], then the pieces and the ks warps' parts are added up
    __syncthreads();
    float* so = reinterpret_cast<float*>(qsm) + warp * (NT * 8 * 16);
#pragma unroll
    for (int n = 0; n < NT; n++) {
        so[(n * 8 + 2 * t) * 16 + g] = acc[n][0];
        so[(n * 8 + 2 * t + 1) * 16 + g] = acc[n][1];
        so[(n * 8 + 2 * t) * 16 + g + 8] = acc[n][2];
        so[(n * 8 + 2 * t + 1) * 16 + g + 8] = acc[n][3];
    }
    __syncthreads();
    const int rows_log2 = 7 - a.ks_log2;
    for (int i = tid; i < mr << rows_log2; i += kQ4Threads) {
        const int r = i >> rows_log2, row = i & (rows - 1), at = blockIdx.x * rows + row;
        if (at >= a.w.rows) continue;
        const float* sp = reinterpret_cast<const float*>(qsm) + ((row >> 4) << a.ks_log2) * (NT * 8 * 16) + (row & 15);
        float v = 0.f;
        for (int k = 0; k < ks; k++)
            for (int j = a.terms - 1; j >= 0; j--) v += sp[k * (NT * 8 * 16) + (r * a.terms + j) * 16];
        st_any(a.out, a.ot, (long long)(r0 + r) * a.ldo + at, v);
    }
}

template <int NT, int P>
static void q4_mma_launch(Context& cx, Q4Args a, cudaStream_t st) {
    const int tiles = (a.w.rows + 15) / 16, gpc = std::min(a.w.group, FHE_Q4_MAX_COLS) / 32;
    // warps enough to keep the loads in flight (8 an SM), but two stages of columns at least for each
    const int chunks = (a.w.cols + 31) / 32;
    a.per = NT * 8 / a.terms;
    a.ks_log2 = 0;
    while (a.ks_log2 < 3 && (tiles << a.ks_log2) < 148 * 8 && chunks >= (4 << a.ks_log2) * kQ4Stage) a.ks_log2++;
    const int step = kQ4Stage << a.ks_log2;
    // as many columns at a time as fit: 512 bytes a chunk and tile of pieces, 512 a chunk for the scales of 8 warps' rows
    a.kb_chunks = std::min((chunks + step - 1) / step * step, kQ4MaxBytes / (512 * (NT + 1)) / step * step);
    a.units = (a.kb_chunks >> a.ks_log2) / P;
    a.group_magic = gpc == 1 ? 0u : (uint32_t)(((1ull << 32) + gpc - 1) / gpc);
    const size_t smem = kQ4RingBytes + (size_t)a.kb_chunks * NT * 512 + (size_t)a.units * kQ4Warps * 64;
    if (smem > 48 * 1024) client_smem<k_q4_mma<NT, P>>(cx);
    const int each = kQ4Warps >> a.ks_log2;
    k_q4_mma<NT, P><<<dim3((tiles + each - 1) / each, (a.m + a.per - 1) / a.per), kQ4Threads, smem, st>>>(a);
    CUDA_CHECK(cudaGetLastError());
    cx.launches++;
}

template <int NT>
static void q4_mma_split(Context& cx, const Q4Args& a, cudaStream_t st) {
    const int gpc = a.w.group / 32;
    if (gpc % 2) q4_mma_launch<NT, 1>(cx, a, st);
    else if (gpc % 4) q4_mma_launch<NT, 2>(cx, a, st);
    else q4_mma_launch<NT, 4>(cx, a, st);
}

static void q4_matvec(Context& cx, Q4Args a, cudaStream_t st) {
    a.terms = a.xt == FHE_F32 ? 3 : a.xt == FHE_F16 ? 2 : 1;
    const long long row = a.ldx * (a.xt == FHE_F32 ? 4 : 2);
    a.wide = (reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(a.m > 1 ? row : 0)) % 16 == 0;
    const int cols = a.m * a.terms;
    if (cols <= 8) q4_mma_split<1>(cx, a, st);
    else if (cols <= 16) q4_mma_split<2>(cx, a, st);
    else if (cols <= 24) q4_mma_split<3>(cx, a, st);
    else q4_mma_split<6>(cx, a, st);
}

// ---- rows of a 4-bit table by token id --------------------------------------------------------
// One warp per row; a token outside the table gives zeros.
__global__ void __launch_bounds__(256) k_q4_rows(const fhe_q4 w, const int64_t* __restrict__ tokens, int m,
                                                 void* __restrict__ out, int ot, long long ldo) {
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= m) return;
    const int64_t t = tokens[r];
    const bool in = t >= 0 && t < w.rows;
    for (int c = lane; c < w.cols; c += 32) {
        float v = 0.f;
        if (in) {
            const int q = w.q[t * w.ldq + c / 2] >> (4 * (c & 1)) & 15;
            v = (float)(q - 8) * ld_any(w.scale, w.scale_type, t * w.lds + c / w.group);
        }
        st_any(out, ot, (long long)r * ldo + c, v);
    }
}

// ---- the choice of a token -----------------------------------------------------------------
// Per row of logits l (NaN counts as -inf), M = max l:
//   z = (l - M) / T (0 where l = M), e = exp(z), weight w = round(2^40 e), a whole number, so that sums of weights do
//   not depend on their order; tokens are ranked by l, equal ones by index;
//   kept: rank < top_k, sum of the weights ranked before < ceil(top_p * the top_k's sum), e >= min_p;
//   S = sum of the kept weights, the token is the first in index order whose running sum passes floor(u S).
constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 2048;      // tokens of one bin that are ranked against each other directly
constexpr float kSampleOne = 1099511627776.f;   // 2^40
// e < 2^-41 rounds to no weight: exp(-29) 2^40 = 0.28, so everything further than 29 T below M is out
constexpr float kSampleReach = 29.f;

struct SampleArgs {
    const void* logits;
    long long ld;
    int type, rows, vocab;
    const float* u;
    const float *temperature, *top_p, *min_p;   // per row, or null: the one value
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int32_t top_k1;
    int64_t* token;
    float* logprob;
};

// larger for what is ranked first: the logit's bits in order, then the lower index
__device__ __forceinline__ uint64_t sample_rank_key(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.f);   // -0 and 0 are equal
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)k << 32 | (0xffffffffu - i);
}

struct SampleRow {
    const void* p;
    int type, v;
    float top, t, bins_per_unit, reach;
    __device__ float x(int i) const {
        const float a = ld_any(p, type, i);
        return a != a ? -INFINITY : a;
    }
    __device__ float z(float a) const { return a == top ? 0.f : __fdiv_rn(a - top, t); }
    __device__ static uint64_t weight(float e) { return __float2ull_rn(e * kSampleOne); }
    __device__ float d(float a) const { return a == top ? 0.f : top - a; }
    __device__ bool counts(float a) const { return a > -INFINITY && d(a) <= reach; }
    __device__ int bin(float a) const { return min(kSampleBins - 1, (int)(d(a) * bins_per_unit)); }
};

template <class T, class F>
__device__ T sample_reduce(T v, F f, T* sh) {
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[threadIdx.x & 31];
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

struct SampleShared {
    uint64_t sum[kSampleBins];
    uint32_t count[kSampleBins];
    uint64_t key[kSampleList], wt[kSampleList];
    uint64_t red[32];
    float redf[32];
    uint32_t n;
    uint64_t got, got_before;
    int at;
};

// The lowest rank key that is still in, among the tokens with keys in [lo, hi], where `want` is a count of tokens (BY_COUNT) or
// a sum of weights: the first token, in rank order, at which the running count or sum reaches `want` (>= 1).  The running
// sum of weights before it goes to *before.  0 if it is never reached.
template <bool BY_COUNT>
__device__ uint64_t sample_select(const SampleRow& row, SampleShared& sh, uint64_t want, uint64_t* before) {
    const int tid = threadIdx.x;
    uint64_t lo = 0, hi = ~0ull, sum_before = 0;
    bool first = true;
    while (true) {
        // histogram of the tokens in [lo, hi]: by distance below the top at first, by rank key after that
        int shift = 0;
        if (!first) {
            const uint64_t range = hi - lo;
            shift = max(0, 64 - __clzll((long long)range) - 11);
        }
        for (int b = tid; b < kSampleBins; b += kSampleThreads) sh.sum[b] = 0, sh.count[b] = 0;
        if (tid == 0) sh.at = -1, sh.n = 0;
        __syncthreads();
        for (int i = tid; i < row.v; i += kSampleThreads) {
            const float a = row.x(i);
            if (!row.counts(a)) continue;
            const uint64_t k = sample_rank_key(a, i);
            if (k < lo || k > hi) continue;
            const int b = first ? row.bin(a) : (int)((hi - k) >> shift);
            atomicAdd(&sh.count[b], 1u);
            atomicAdd((unsigned long long*)&sh.sum[b], (unsigned long long)row.weight(expf(row.z(a))));
        }
        __syncthreads();
        if (tid == 0) {
            uint64_t run = 0, s = sum_before;
            for (int b = 0; b < kSampleBins; b++) {
                const uint64_t now = BY_COUNT ? sh.count[b] : sh.sum[b];
                if (run + now >= want) { sh.at = b; sh.got = run; sh.got_before = s; break; }
                run += now;
                s += sh.sum[b];
            }
            if (sh.at < 0) sh.got_before = s;
        }
        __syncthreads();
        const int at = sh.at;
        sum_before = sh.got_before;
        if (at < 0) { *before = sum_before; return 0; }
        want -= sh.got;
        const uint32_t n = sh.count[at];
        if (n <= kSampleList) {
            for (int i = tid; i < row.v; i += kSampleThreads) {
                const float a = row.x(i);
                if (!row.counts(a)) continue;
                const uint64_t k = sample_rank_key(a, i);
                if (k < lo || k > hi) continue;
                const int b = first ? row.bin(a) : (int)((hi - k) >> shift);
                if (b != at) continue;
                const uint32_t j = atomicAdd(&sh.n, 1u);
                sh.key[j] = k;
                sh.wt[j] = row.weight(expf(row.z(a)));
            }
            __syncthreads();
            // the list's own order: each token sums what is ranked before it
            for (uint32_t j = tid; j < n; j += kSampleThreads) {
                const uint64_t k = sh.key[j];
                uint64_t c = 0, s = 0;
                for (uint32_t l = 0; l < n; l++)
                    if (sh.key[l] > k) { c++; s += sh.wt[l]; }
                const uint64_t run = BY_COUNT ? c : s, own = BY_COUNT ? 1 : sh.wt[j];
                if (run < want && run + own >= want) { sh.got = k; sh.got_before = sum_before + s; }
            }
            __syncthreads();
            *before = sh.got_before;
            const uint64_t r = sh.got;
            __syncthreads();
            return r;
        }
        // too many: their own range of rank keys, in finer bins
        uint64_t a0 = ~0ull, a1 = 0;
        for (int i = tid; i < row.v; i += kSampleThreads) {
            const float a = row.x(i);
            if (!row.counts(a)) continue;
            const uint64_t k = sample_rank_key(a, i);
            if (k < lo || k > hi) continue;
            const int b = first ? row.bin(a) : (int)((hi - k) >> shift);
            if (b == at) a0 = min(a0, k), a1 = max(a1, k);
        }
        lo = sample_reduce(a0, [](uint64_t p, uint64_t q) { return min(p, q); }, sh.red);
        hi = sample_reduce(a1, [](uint64_t p, uint64_t q) { return max(p, q); }, sh.red);
        first = false;
    }
}

__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t ssm[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(ssm);
    const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    SampleRow row;
    row.p = static_cast<const uint8_t*>(a.logits) + (long long)r * a.ld * (a.type == FHE_F32 ? 4 : 2);
    row.type = a.type;
    row.v = a.vocab;
    float t = a.temperature ? a.temperature[r] : a.temperature1;
    float p = a.top_p ? a.top_p[r] : a.top_p1;
    float mp = a.min_p ? a.min_p[r] : a.min_p1;
    int64_t k = a.top_k ? a.top_k[r] : a.top_k1;
    mp = mp > 0.f ? fminf(mp, 1.f) : 0.f;   // a NaN in the array: off
    if (!(t > 0.f)) t = 1.f, k = 1;
    float top = -INFINITY, low = INFINITY;
    for (int i = tid; i < row.v; i += kSampleThreads) {
        const float x = row.x(i);
        top = fmaxf(top, x);
        if (x > -INFINITY) low = fminf(low, x);
    }
    row.top = top = sample_reduce(top, [](float x, float y) { return fmaxf(x, y); }, sh.redf);
    low = sample_reduce(low, [](float x, float y) { return fminf(x, y); }, sh.redf);
    if (top == -INFINITY) {
        if (tid == 0) a.token[r] = -1, a.logprob[r] = -INFINITY;
        return;
    }
    row.t = t;
    row.reach = kSampleReach * t;
    const float span = fminf(row.reach, top - low);
    row.bins_per_unit = span > 0.f ? fminf(kSampleBins / span, 1e30f) : 0.f;

    uint64_t bound = 0, before;
    const bool by_p = p < 1.f;
    if (k > 0 && k < row.v) bound = sample_select<true>(row, sh, k, &before);
    if (by_p) {
        uint64_t s = 0;
        for (int i = tid; i < row.v; i += kSampleThreads) {
            const float x = row.x(i);
            if (row.counts(x) && sample_rank_key(x, i) >= bound) s += row.weight(expf(row.z(x)));
        }
        s = sample_reduce(s, [](uint64_t x, uint64_t y) { return x + y; }, sh.red);
        const double want = ceil((double)p * (double)s);
        const uint64_t b = sample_select<false>(row, sh, want > 1.0 ? (uint64_t)want : 1, &before);
        bound = max(bound, b);
    }
    // the kept weights of each warp's stretch of tokens
    const int per = (row.v + kSampleWarps - 1) / kSampleWarps, i0 = min(row.v, warp * per), i1 = min(row.v, i0 + per);
    auto kept = [&](int i) -> uint64_t {
        const float x = row.x(i);
        if (!row.counts(x) || sample_rank_key(x, i) < bound) return 0;
        const float e = expf(row.z(x));
        return e >= mp ? row.weight(e) : 0;
    };
    uint64_t mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += kept(i);
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) sh.red[warp] = mine;
    __syncthreads();
    uint64_t total = 0, start = 0;
    for (int w = 0; w < kSampleWarps; w++) {
        if (w == warp) start = total;
        total += sh.red[w];
    }
    const float u = fminf(fmaxf(a.u[r], 0.f), 1.f);
    uint64_t target = (uint64_t)((double)u * (double)total);
    if (target >= total) target = total - 1;
    if (target < start || target >= start + mine) return;
    for (int i = i0; i < i1; i += 32) {
        const uint64_t w = i + lane < i1 ? kept(i + lane) : 0;
        uint64_t run = w;
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, start + run > target);
        if (past) {
            if (lane == __ffs(past) - 1) {
                a.token[r] = i + lane;
                a.logprob[r] = row.z(row.x(i + lane)) - (float)log((double)total / (double)kSampleOne);
            }
            return;
        }
        start += __shfl_sync(0xffffffffu, run, 31);
    }
}

}  // namespace fhe

// ---- the C ABI --------------------------------------------------------------------------------
namespace {

int client_type_bytes(int type, const char* what) {
    if (type != FHE_F32 && type != FHE_F16 && type != FHE_BF16)
        throw fhe::Error(std::string(what) + ": unknown type", FHE_ERR_ARG);
    return type == FHE_F32 ? 4 : 2;
}

// device memory of the context's GPU, aligned to `align` bytes
void client_ptr(const fhe::Context& c, const void* p, size_t align, const char* what) {
    cudaPointerAttributes at{};
    if (!p) throw fhe::Error(std::string(what) + " is null", FHE_ERR_ARG);
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        throw fhe::Error(std::string("cannot query ") + what, FHE_ERR_ARG);
    }
    const bool dev = at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged;
    if (!dev || at.device != c.device)
        throw fhe::Error(std::string(what) + " is not device memory of the context's GPU", FHE_ERR_ARG);
    if (reinterpret_cast<uintptr_t>(p) % align)
        throw fhe::Error(std::string(what) + " is not " + std::to_string(align) + "-byte aligned", FHE_ERR_ARG);
}

void client_table(const fhe::Context& c, const fhe_q4* w) {
    REQUIRE(w, "null argument");
    REQUIRE(w->rows >= 0 && w->cols >= 1 && w->cols <= FHE_Q4_MAX_COLS,
            "q4 table: rows >= 0 and cols in 1..FHE_Q4_MAX_COLS");
    REQUIRE(w->group >= 32 && w->group % 32 == 0, "q4 table: the group is a multiple of 32 columns");
    REQUIRE(w->ldq % 16 == 0 && w->ldq >= ((long long)w->cols + 31) / 32 * 16,
            "q4 table: rows are padded to a multiple of 16 bytes (32 columns)");
    REQUIRE(w->lds >= ((long long)w->cols + w->group - 1) / w->group, "q4 table: a scale for each group of a row");
    const int sb = client_type_bytes(w->scale_type, "q4 scales");
    if (!w->rows) return;
    client_ptr(c, w->q, 16, "q4 table");
    client_ptr(c, w->scale, sb, "q4 scales");
}

cudaStream_t client_stream(fhe_ctx* cx, void* stream) {
    CUDA_CHECK(cudaSetDevice(cx->cx.device));
    return stream ? static_cast<cudaStream_t>(stream) : cx->cx.stream;
}

}  // namespace

extern "C" int fhe_q4_matvec(fhe_ctx* cx, const fhe_q4* w, const void* x, int x_type, long long ldx, int m, void* out,
                             int out_type, long long ldo, void* stream) {
    return guard([&] {
        REQUIRE(cx, "null argument");
        client_table(cx->cx, w);
        const int xb = client_type_bytes(x_type, "x"), ob = client_type_bytes(out_type, "out");
        REQUIRE(m >= 0, "m is negative");
        REQUIRE(ldx >= w->cols || m <= 1, "x: rows are shorter than the table's columns");
        REQUIRE(ldo >= w->rows || m <= 1, "out: rows are shorter than the table's rows");
        if (m == 0 || w->rows == 0) return;
        client_ptr(cx->cx, x, xb, "x");
        client_ptr(cx->cx, out, ob, "out");
        cudaStream_t st = client_stream(cx, stream);
        fhe::q4_matvec(cx->cx, fhe::Q4Args{*w, x, x_type, 0, m, ldx, out, out_type, ldo, 0, 0, 0, 0, 0, 0}, st);
    });
}

extern "C" int fhe_q4_rows(fhe_ctx* cx, const fhe_q4* w, const int64_t* tokens, int m, void* out, int out_type,
                           long long ldo, void* stream) {
    return guard([&] {
        REQUIRE(cx, "null argument");
        client_table(cx->cx, w);
        const int ob = client_type_bytes(out_type, "out");
        REQUIRE(m >= 0, "m is negative");
        REQUIRE(ldo >= w->cols || m <= 1, "out: rows are shorter than the table's columns");
        if (m == 0) return;
        client_ptr(cx->cx, tokens, 8, "tokens");
        client_ptr(cx->cx, out, ob, "out");
        cudaStream_t st = client_stream(cx, stream);
        fhe::k_q4_rows<<<(m + 7) / 8, 256, 0, st>>>(*w, tokens, m, out, out_type, ldo);
        CUDA_CHECK(cudaGetLastError());
        cx->cx.launches++;
    });
}

extern "C" int fhe_sample(fhe_ctx* cx, const fhe_sample_cfg* cfg, const void* logits, int type, long long ld, int rows,
                          int vocab, const float* u, int64_t* token, float* logprob, void* stream) {
    return guard([&] {
        REQUIRE(cx && cfg, "null argument");
        const int b = client_type_bytes(type, "logits");
        REQUIRE(rows >= 0 && vocab >= 1, "sample: rows >= 0 and vocab >= 1");
        REQUIRE(vocab <= FHE_SAMPLE_MAX_VOCAB, "sample: the vocabulary is above FHE_SAMPLE_MAX_VOCAB");
        REQUIRE(ld >= vocab || rows <= 1, "logits: rows are shorter than the vocabulary");
        if (!cfg->temperature) REQUIRE(cfg->temperature_all >= 0.f && cfg->temperature_all <= 1e30f,
                                       "sample: temperature is a finite number >= 0");
        if (!cfg->top_k) REQUIRE(cfg->top_k_all >= 0, "sample: top_k >= 0 (0: off)");
        if (!cfg->top_p) REQUIRE(cfg->top_p_all > 0.f && cfg->top_p_all <= 1.f, "sample: top_p in (0, 1]");
        if (!cfg->min_p) REQUIRE(cfg->min_p_all >= 0.f && cfg->min_p_all <= 1.f, "sample: min_p in [0, 1]");
        if (rows == 0) return;
        client_ptr(cx->cx, logits, b, "logits");
        client_ptr(cx->cx, u, 4, "u");
        client_ptr(cx->cx, token, 8, "token");
        client_ptr(cx->cx, logprob, 4, "logprob");
        if (cfg->temperature) client_ptr(cx->cx, cfg->temperature, 4, "temperature");
        if (cfg->top_k) client_ptr(cx->cx, cfg->top_k, 4, "top_k");
        if (cfg->top_p) client_ptr(cx->cx, cfg->top_p, 4, "top_p");
        if (cfg->min_p) client_ptr(cx->cx, cfg->min_p, 4, "min_p");
        cudaStream_t st = client_stream(cx, stream);
        fhe::SampleArgs a{logits, ld, type, rows, vocab, u, cfg->temperature, cfg->top_p, cfg->min_p, cfg->top_k,
                          cfg->temperature_all, cfg->top_p_all, cfg->min_p_all, cfg->top_k_all, token, logprob};
        const size_t smem = sizeof(fhe::SampleShared);
        fhe::client_smem<fhe::k_sample>(cx->cx);
        fhe::k_sample<<<rows, fhe::kSampleThreads, smem, st>>>(a);
        CUDA_CHECK(cudaGetLastError());
        cx->cx.launches++;
    });
}
