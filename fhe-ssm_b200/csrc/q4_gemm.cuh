// q4_gemm.cuh -- products of several rows with a 4-bit table on the 5th-generation tensor cores (tcgen05).
//
//     out[r][i] = sum_g s[i][g] sum_{c in g} (q[i][c] - 8) x[r][c]
//
// The inner sum is a 16-bit tensor-core product of whole numbers with x; the scale is applied to it in float32, as it
// leaves tensor memory.  x is carried in float16, scaled by a power of two of its row's maximum: float16 and bfloat16 as they
// are, float32 as two pieces of 11 bits, the one rounding before the float32 sums.  (The table in bfloat16 takes 11
// instructions for 8 values to unpack, in float16 9, and the issue slots bound this kernel.)
//
// k_q4_pack writes x's operand as the shared-memory image of its chunks of columns; k_q4_gemm starts while it runs
// (programmatic dependent launch) and waits for it where it first loads the image.
//
// Per block of k_q4_gemm: up to 4 tiles of 128 table rows (lanes of tensor memory) x N rows of x (its columns).  Roles:
//   warps 0-7    drain: accumulators of a chunk of columns -> registers, times the rows' scales; output
//   warps 8-15   two groups in turn: table bytes (cp.async ring) -> 16-bit operands in tensor memory
//   warp 16      issues the products
//   warp 17      loads x's chunks (bulk copies)
//   warps 18-19  scales -> shared memory, a tile ahead of the drain
// The table operand goes to tensor memory and not to shared memory, whose bandwidth the products would then share with
// its writes: 16 KB written and 16 KB a piece read for each 128 x 64 tile, four times the time of the product itself.
// x's operand stays in shared memory for as many columns as fit (a range); the tiles pass over it one after the other, and
// between ranges a tile's sums wait in tensor memory, so the drain needs registers for one tile only.
//
// 64 float32 rows on 50,304 x 1,024 at groups of 64 take 24.2 us, bfloat16 rows 20.8 (316 TFLOP/s; 19% of cuBLAS's bfloat16
// rate, 1.9 TB/s), on 65,536 x 1,024 25.1, 16 rows on 50,304 x 1,024 18.0.  About 8 us are the two launches, the operand's image,
// the first tile's way through the roles and the last output; then 0.25 to 0.3 us for each 128 x 64 of the table, which is the
// unpacking's and the drain's instructions: 55% of the issue slots over the whole kernel, with its waits between roles.
//
// Included by client.cu inside namespace fhe.

constexpr int kQgThreads = 640;
constexpr int kQgRowsMax = 512;               // table rows of a block
constexpr int kQgStages = 4;                  // 128 rows x 128 columns of table bytes each, for each group
constexpr int kQgStageBytes = 128 * 64;
constexpr int kQgAMax = 4, kQgDMax = 4;       // operand (a job each) and accumulator (a chunk each) slots in tensor memory
constexpr int kQgSlotsMax = 8;                // jobs of x's operand
constexpr int kQgXBytes = 131072;             // shared memory for them
// A wait that has nothing to wait for costs 110 cycles, a commit 46 (measured alone), so they are few: operands change hands by
// the job of 128 columns, and one wait of the products' warp sees to several barriers, a lane each.  (Waits with a sleep
// time as a hint wake later: the whole kernel took 1.3 times as long with 20 us.)
constexpr int kQgWaits = 1 << 22;             // every wait is bounded: some seconds

struct QgBars {
    uint64_t a_full[kQgAMax], a_empty[kQgAMax], d_full[kQgDMax], d_empty[kQgDMax], x_full[kQgSlotsMax], x_empty[kQgSlotsMax],
        s_full[2], s_empty[2], p_full, end;
    uint32_t tmem;
    int dead;      // a wait ran out: the output is NaN
};

struct QgArgs {
    fhe_q4 w;
    const void* x;
    int m;
    long long ldx;
    void* out;
    int ot;
    long long ldo;
    int wide;         // rows of x start on 16-byte boundaries
    int block_rows;   // table rows of a block
    int slots;        // jobs of a range
    int jobs;         // jobs of all columns, 128 each
    int groups;       // most groups that a range meets
    int part_jobs;    // jobs of a part (blockIdx.z)
    float* parts;     // [part][row of x][table row], or null: one part, which writes the output
    int run;          // chunks that one accumulator takes before the scale is applied
    uint8_t* image;   // x's operand [tile of N rows][chunk][piece], then the rows' powers
    float* powers;    // 2^p, by which the rows' sums are multiplied
    int waits;        // tries of the waits for a free slot (kQgWaits, or what the context's q4_waits says)
};

__device__ __forceinline__ void qg_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc_smem(bar)), "r"(count));
}
__device__ __forceinline__ void qg_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc_smem(bar)) : "memory");
}
__device__ __forceinline__ void qg_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tc_smem(bar)) : "memory");
}
__device__ __forceinline__ bool qg_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(tc_smem(bar)), "r"(parity)
        : "memory");
    return ok;
}
// Waits until the phase of the given parity has passed.  False: this wait ran out, or another one of the block has (dead).  Whoever
// writes operands, issues products or starts copies then stops, so that nothing is written that may still be read and no barrier
// counts a copy twice.  The drain goes on without a test for each chunk, which cost the 64-row products 20 to 35% of their time: it
// reads and lets go of accumulators and scales, whose sums, for all who still read them, are written out as NaN.  (A number of tries that is not a constant costs the products'
// warp 5% at groups of 32, so only the waits for a free slot have one.)
__device__ __forceinline__ bool qg_wait(uint64_t* bar, uint32_t parity, QgBars* b, int tries) {
    if (qg_try(bar, parity)) return true;
    for (int it = 0; it < tries; it++) {
        if (qg_try(bar, parity)) return true;
        if ((it & 63) == 63 && *(volatile int*)&b->dead) return false;
    }
    *(volatile int*)&b->dead = 1;
    return false;
}
// the same by a warp, whose lanes stay together
__device__ __forceinline__ bool qg_wait_warp(uint64_t* bar, uint32_t parity, QgBars* b, int tries) {
    return __all_sync(0xffffffffu, qg_wait(bar, parity, b, tries));
}

// kind::f16, D float32, both operands float16 and K-major, M = 128, N = n
__device__ constexpr uint32_t qg_idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }
__device__ __forceinline__ void qg_mma(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(acc), "r"(0), "r"(0), "r"(0), "r"(0));
}

#define QG_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define QG_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// CNT columns of the warp's 32 lanes
template <int CNT>
__device__ __forceinline__ void qg_ld(uint32_t t, uint32_t* v) {
    if constexpr (CNT == 32)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : QG_R8(v, 0), QG_R8(v, 8), QG_R8(v, 16), QG_R8(v, 24)
            : "r"(t));
    else if constexpr (CNT == 16)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : QG_R8(v, 0), QG_R8(v, 8)
            : "r"(t));
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : QG_R8(v, 0) : "r"(t));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
template <int CNT>
__device__ __forceinline__ void qg_st(uint32_t t, const uint32_t* v) {
    if constexpr (CNT == 32)
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(t),
            QG_W8(v, 0), QG_W8(v, 8), QG_W8(v, 16), QG_W8(v, 24)
            : "memory");
    else if constexpr (CNT == 16)
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16};" ::"r"(t),
            QG_W8(v, 0), QG_W8(v, 8)
            : "memory");
    else
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(t), QG_W8(v, 0)
                     : "memory");
}

// 8 values of 4 bits -> float16 pairs (0,4), (1,5), (2,6), (3,7) of q - 8.  0x6400 is 1024, whose last bits count in ones: 1024 + q,
// or 1024 + 16 q from the high half of a byte.
__device__ __forceinline__ void qg_unpack(uint32_t w, uint32_t* p) {
    const __half2 off = __float2half2_rn(1032.f), by = __float2half2_rn(0.0625f), low = __float2half2_rn(-72.f);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t a = (w & 0x000f000fu) | 0x64006400u, b = (w & 0x00f000f0u) | 0x64006400u;
        const __half2 u = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
        const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&b), by, low);
        p[i] = *reinterpret_cast<const uint32_t*>(&u);
        p[i + 1] = *reinterpret_cast<const uint32_t*>(&v);
        w >>= 8;
    }
}
__device__ __forceinline__ uint64_t qg_pack2(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
// two float32 multiply-adds
__device__ __forceinline__ uint64_t qg_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

__device__ __forceinline__ void qg_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void qg_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void qg_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <int KC>
__host__ __device__ constexpr uint32_t qg_sbo() { return KC / 8 * 128; }   // bytes of 8 rows of a chunk of x's operand

// x -> operand image.  One block per row; a thread takes 8 columns, in the order of qg_unpack's pairs.
template <int N, int KC, class XT>
__global__ void __launch_bounds__(128) k_q4_pack(const QgArgs a) {
    constexpr bool kF32 = std::is_same<XT, float>::value, kF16 = std::is_same<XT, __half>::value;
    constexpr int kPieces = kF32 ? 2 : 1, kPieceBytes = N * KC * 2;
    pdl_trigger();
    const int r = blockIdx.x, n = r % N, units = a.jobs * 16;
    uint8_t* to = a.image + (size_t)(r / N) * a.jobs * (128 / KC) * kPieces * kPieceBytes + (n >> 3) * qg_sbo<KC>() + (n & 7) * 16;
    const auto load = [&](int u, XT* v) {
        const int k = u * 8;
        const XT* src = static_cast<const XT*>(a.x) + r * a.ldx + k;
        if (r < a.m && a.wide && k + 8 <= a.w.cols) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(XT) / 2; j++) reinterpret_cast<uint4*>(v)[j] = reinterpret_cast<const uint4*>(src)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = r < a.m && k + j < a.w.cols ? src[j] : XT(0.f);
        }
    };
    const auto pair = [](__half x, __half y) { return (uint32_t)__half_as_ushort(x) | (uint32_t)__half_as_ushort(y) << 16; };
    __align__(16) XT v[8];
    load(threadIdx.x, v);
    float up = 1.f;
    if constexpr (!kF16) {
        // the row's largest finite magnitude maps to 2^14 .. 2^15; a value under 2^-16 of it is held to 2^-39 of it
        uint32_t most = 0;
        const auto see = [&](const XT* u) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t bits = __float_as_uint(q4_float(u[j])) & 0x7fffffffu;
                most = max(most, bits < 0x7f800000u ? bits : 0u);
            }
        };
        see(v);
        for (int u = threadIdx.x + 128; u < units; u += 128) {
            __align__(16) XT w[8];
            load(u, w);
            see(w);
        }
        __shared__ uint32_t sm[4];
        most = __reduce_max_sync(0xffffffffu, most);
        if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = most;
        __syncthreads();
        const int e = max(15, (int)(max(max(sm[0], sm[1]), max(sm[2], sm[3])) >> 23));
        up = __uint_as_float((uint32_t)(268 - e) << 23);
        if (threadIdx.x == 0) a.powers[r] = __uint_as_float((uint32_t)(e - 14) << 23);
    } else if (threadIdx.x == 0) {
        a.powers[r] = 1.f;
    }
    for (int u = threadIdx.x; u < units; u += 128) {
        if (u != threadIdx.x) load(u, v);
        uint8_t* dst = to + (size_t)(u / (KC / 8)) * kPieces * kPieceBytes + u % (KC / 8) * 128;
        __half h[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (kF16) h[j] = v[j];
            else h[j] = __float2half_rn(q4_float(v[j]) * up);
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(pair(h[0], h[4]), pair(h[1], h[5]), pair(h[2], h[6]), pair(h[3], h[7]));
        if constexpr (kF32) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // what the first piece leaves; an infinity or NaN is all in the first
                const float f = __half2float(h[j]), rest = v[j] * up - f;
                h[j] = __float2half_rn(fabsf(f) < INFINITY ? rest : 0.f);
            }
            *reinterpret_cast<uint4*>(dst + kPieceBytes) =
                make_uint4(pair(h[0], h[4]), pair(h[1], h[5]), pair(h[2], h[6]), pair(h[3], h[7]));
        }
    }
}

// N rows of x (16, 32 or 64) in kPieces pieces, KC columns a chunk (64, or 32 where the group is no multiple of 64)
template <int N, int KC, int kPieces>
__global__ void __launch_bounds__(kQgThreads, 1) k_q4_gemm(const QgArgs a, unsigned int* err) {
    constexpr int kItems = 128 / KC;                    // chunks of a job
    constexpr int kPieceBytes = N * KC * 2, kChunkBytes = kPieceBytes * kPieces, kSlotBytes = kChunkBytes * kItems;
    extern __shared__ __align__(1024) uint8_t gsm[];
    uint8_t* ring = gsm;
    uint8_t* xs = gsm + 2 * kQgStages * kQgStageBytes;
    float* scales = reinterpret_cast<float*>(xs + (size_t)a.slots * kSlotBytes);   // [2][group of the range][128 rows]
    float* powers = scales + 2 * a.groups * 128;                                    // [N]
    QgBars* bars = reinterpret_cast<QgBars*>(powers + N);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * a.block_rows, row1 = min(a.w.rows, row0 + a.block_rows), tiles = (row1 - row0 + 127) / 128;
    const int x0 = blockIdx.y * N;
    const int job0 = blockIdx.z * a.part_jobs, all_jobs = min(a.part_jobs, a.jobs - job0);
    const int ranges = (all_jobs + a.slots - 1) / a.slots;
    const auto range_jobs = [&](int kr) { return min(a.slots, all_jobs - kr * a.slots); };
    if (a.parts) pdl_trigger();   // k_q4_sum, which waits for this kernel
    // tensor memory: the tiles' sums (several ranges only), accumulators, operands.  Two or four operand slots: a slot is
    // always filled by the same of the two groups, which so cannot get more than the one phase that a parity tells ahead of it.
    const uint32_t dcol = ranges > 1 ? tiles * N : 0, nd = min((uint32_t)kQgDMax, (384 - dcol) / N), acol = dcol + nd * N;
    const int na = acol <= 256 ? 4 : 2;

    if (tid == 0) {
        for (int i = 0; i < kQgAMax; i++) qg_init(&bars->a_full[i], 4), qg_init(&bars->a_empty[i], 1);
        for (int i = 0; i < kQgDMax; i++) qg_init(&bars->d_full[i], 1), qg_init(&bars->d_empty[i], 8);
        for (int i = 0; i < a.slots; i++) qg_init(&bars->x_full[i], 1), qg_init(&bars->x_empty[i], 1);
        for (int i = 0; i < 2; i++) qg_init(&bars->s_full[i], 64), qg_init(&bars->s_empty[i], 8);
        qg_init(&bars->p_full, 1);
        qg_init(&bars->end, 1);
        bars->dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&bars->tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tm = bars->tmem, lanes = (uint32_t)(32 * (warp & 3)) << 16;

    if (warp < 8) {
        // ---- drain: row = lane of the tile, half of the columns
        constexpr int kC = N / 2;
        const int half = warp >> 2, per_group = a.w.group / (KC * a.run);
        uint32_t slot = 0, phase = 0, tile = 0;
        for (int kr = 0; kr < ranges; kr++) {
            const int drains = range_jobs(kr) * kItems / a.run;
            for (int b = 0; b < tiles; b++, tile++) {
                const int row = row0 + b * 128 + (warp & 3) * 32 + lane;
                int left = per_group - (job0 + kr * a.slots) * kItems / a.run % per_group;
                const float* sp = scales + (tile & 1) * a.groups * 128 + (warp & 3) * 32 + lane;
                qg_wait(&bars->s_full[tile & 1], tile >> 1 & 1, bars, kQgWaits);
                uint64_t acc2[kC / 2];
#pragma unroll
                for (int j = 0; j < kC / 2; j++) acc2[j] = 0;
                for (int c = 0; c < drains; c++) {
                    const float s = *sp;
                    if (--left == 0) left = per_group, sp += 128;
                    qg_wait(&bars->d_full[slot], phase, bars, kQgWaits);
                    __syncwarp();
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    uint32_t v[kC];
                    qg_ld<kC>(tm + dcol + slot * N + half * kC + lanes, v);
                    asm volatile("tcgen05.fence::before_thread_sync;");
                    __syncwarp();
                    if (lane == 0) qg_arrive(&bars->d_empty[slot]);
                    const uint64_t s2 = qg_pack2(__float_as_uint(s), __float_as_uint(s));
#pragma unroll
                    for (int j = 0; j < kC / 2; j++) acc2[j] = qg_fma2(s2, qg_pack2(v[2 * j], v[2 * j + 1]), acc2[j]);
                    if (++slot == nd) slot = 0, phase ^= 1;
                }
                float acc[kC];
#pragma unroll
                for (int j = 0; j < kC; j++) acc[j] = __uint_as_float((uint32_t)(acc2[j / 2] >> (32 * (j & 1))));
                __syncwarp();
                if (lane == 0) qg_arrive(&bars->s_empty[tile & 1]);
                const uint32_t keep = tm + b * N + half * kC + lanes;
                if (kr) {
                    uint32_t v[kC];
                    qg_ld<kC>(keep, v);
#pragma unroll
                    for (int j = 0; j < kC; j++) acc[j] += __uint_as_float(v[j]);
                }
                if (kr + 1 < ranges) {
                    qg_st<kC>(keep, reinterpret_cast<const uint32_t*>(acc));
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    continue;
                }
                const int r0 = x0 + half * kC, nr = min(kC, a.m - r0);
                qg_wait(&bars->p_full, 0, bars, kQgWaits);
                if (*(volatile int*)&bars->dead) {
#pragma unroll
                    for (int j = 0; j < kC; j++) acc[j] = __int_as_float(0x7fffffff);
                }
#pragma unroll
                for (int j = 0; j < kC; j += 4) {
                    const float4 p = *reinterpret_cast<const float4*>(powers + half * kC + j);
                    acc[j] *= p.x, acc[j + 1] *= p.y, acc[j + 2] *= p.z, acc[j + 3] *= p.w;
                }
                if (row >= row1) continue;
                const auto store = [&](auto* out, long long ldo) {
                    out += r0 * ldo + row;
                    if (nr >= kC) {
#pragma unroll
                        for (int j = 0; j < kC; j++, out += ldo) qg_store(out, acc[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < kC; j++, out += ldo)
                            if (j < nr) qg_store(out, acc[j]);
                    }
                };
                if (a.parts) store(a.parts + (long long)blockIdx.z * a.m * a.w.rows, a.w.rows);
                else if (a.ot == FHE_F32) store(static_cast<float*>(a.out), a.ldo);
                else if (a.ot == FHE_F16) store(static_cast<__half*>(a.out), a.ldo);
                else store(static_cast<__nv_bfloat16*>(a.out), a.ldo);
            }
        }
    } else if (warp < 16) {
        // ---- the table: jobs of 128 rows x 128 columns, every second one
        const int grp = (warp >> 2) - 2, t = tid & 127;
        uint8_t* my = ring + grp * kQgStages * kQgStageBytes;
        const int units = (a.w.cols + 31) / 32;   // 16-byte units of a row
        const int jobs = tiles * all_jobs;
        // the job to fetch next; a thread copies the same 16-byte unit of 4 rows
        int fkr = 0, fb = 0, fc = grp, fn = range_jobs(0), fat = 0;
        const long long ld32 = 32 * a.w.ldq;
        const uint8_t* fsrc = a.w.q + (row0 + (t >> 2)) * a.w.ldq + job0 * 64 + (t & 3) * 16;
        const uint32_t fdst = tc_smem(my) + (t >> 2) * 64 + (((t & 3) ^ (t >> 3 & 3)) << 4);
        const auto fetch = [&]() {
            while (fc >= fn) {
                fc -= fn;
                if (++fb < tiles) {
                    fsrc += 4 * ld32;
                } else if (++fkr < ranges) {
                    fsrc += a.slots * 64 - (tiles - 1) * 4 * ld32;
                    fb = 0;
                    fn = range_jobs(fkr);
                } else {
                    fn = 1 << 30;   // no more
                }
            }
            if (fkr < ranges && (job0 + fkr * a.slots + fc) * 4 + (t & 3) < units) {
                const uint8_t* src = fsrc + fc * 64;
                const int row = row0 + fb * 128 + (t >> 2);
#pragma unroll
                for (int i = 0; i < 4; i++, src += ld32)
                    if (row + 32 * i < row1)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(fdst + fat * kQgStageBytes + i * 2048), "l"(src)
                                     : "memory");
            }
            fc += 2;
            fat = (fat + 1) % kQgStages;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int s = 0; s < kQgStages - 1; s++) fetch();
        uint32_t slot = grp, phase = 1;
        bool live = true;   // after a wait that ran out the warp still meets the others at their barrier, and only there
        for (int j = grp, s = 0; j < jobs; j += 2, s++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kQgStages - 2) : "memory");
            // all copies of the stage are there; the one before it is read
            if (grp == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
            else asm volatile("bar.sync 2, 128;" ::: "memory");
            fetch();
            if (!live) continue;
            const uint8_t* st = my + (s % kQgStages) * kQgStageBytes + t * 64;
#pragma unroll 1
            for (int h = 0; h < kItems; h++) {
                uint32_t v[KC / 2];
#pragma unroll
                for (int q = 0; q < KC / 32; q++) {
                    const uint4 u = *reinterpret_cast<const uint4*>(st + (((h * (KC / 32) + q) ^ (t >> 1 & 3)) << 4));
                    qg_unpack(u.x, v + q * 16);
                    qg_unpack(u.y, v + q * 16 + 4);
                    qg_unpack(u.z, v + q * 16 + 8);
                    qg_unpack(u.w, v + q * 16 + 12);
                }
                if (h == 0) {
                    if (!qg_wait_warp(&bars->a_empty[slot], phase, bars, a.waits)) {
                        live = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;");
                }
                qg_st<KC / 2>(tm + acol + slot * 64 + h * (KC / 2) + lanes, v);
            }
            if (!live) continue;
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0) qg_arrive(&bars->a_full[slot]);
            if ((slot += 2) >= na) slot = grp, phase ^= 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 16) {
        // ---- products: one lane issues them, the warp stays together
        constexpr uint32_t idesc = qg_idesc(N);
        uint32_t elected;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(elected));
        const uint32_t base = __reduce_or_sync(0xffffffffu, tm);   // the same in all lanes, as the compiler now sees
        const uint64_t xdesc = tc_desc(tc_smem(xs), 128, qg_sbo<KC>());
        uint32_t i = 0, aphase = 0, slot = 0, dphase = 1;
        const auto issue = [&]() {
            for (int kr = 0; kr < ranges; kr++) {
                const int n = range_jobs(kr);
                for (int b = 0; b < tiles; b++)
                    for (int c = 0; c < n; c++) {
                        const uint32_t at = base + acol + i * 64;
                        const uint64_t xd = xdesc + (uint32_t)(c * kSlotBytes >> 4);
#pragma unroll
                        for (int h = 0; h < kItems; h += 2) {   // two chunks at a time, of one accumulator or two
                            const bool wrap = slot + 1 == nd;
                            const uint32_t slot1 = a.run == 2 ? slot : wrap ? 0 : slot + 1, phase1 = a.run == 1 && wrap ? dphase ^ 1 : dphase;
                            uint64_t* bar = lane == 0   ? &bars->a_full[i]
                                            : lane == 1 ? &bars->d_empty[slot]
                                            : lane == 2 ? &bars->d_empty[slot1]
                                                        : &bars->x_full[c];
                            if (!qg_wait_warp(bar, lane == 0 ? aphase : lane == 1 ? dphase : lane == 2 ? phase1 : kr & 1, bars,
                                              kQgWaits))
                                return;
                            asm volatile("tcgen05.fence::after_thread_sync;");
                            if (elected) {
#pragma unroll
                                for (int g = 0; g < 2; g++) {
#pragma unroll
                                    for (int p = 0; p < kPieces; p++)
#pragma unroll
                                        for (int ks = 0; ks < KC / 16; ks++)
                                            qg_mma(base + dcol + (g ? slot1 : slot) * N, at + (h + g) * (KC / 2) + ks * 8,
                                                   xd + (((h + g) * kChunkBytes + p * kPieceBytes + ks * 256) >> 4), idesc,
                                                   p + ks > 0 || (g && a.run == 2));
                                    if (g || a.run == 1) qg_commit(&bars->d_full[g ? slot1 : slot]);
                                }
                                if (h + 2 == kItems) {
                                    qg_commit(&bars->a_empty[i]);
                                    if (b == tiles - 1 && kr + 1 < ranges) qg_commit(&bars->x_empty[c]);
                                }
                            }
                            __syncwarp();
                            slot = slot1;
                            dphase = phase1;
                            if (++slot == nd) slot = 0, dphase ^= 1;
                        }
                        if (++i == na) i = 0, aphase ^= 1;
                    }
            }
        };
        issue();
        if (elected) {
            qg_commit(&bars->end);   // all products, before tensor memory is given back
            for (int it = 0; it < kQgWaits && !qg_try(&bars->end, 0); it++) {}
        }
        __syncwarp();
    } else if (warp == 17) {
        // ---- x
        pdl_wait();
        for (int j = lane; j < N; j += 32) powers[j] = a.powers[x0 + j];
        __syncwarp();
        if (lane == 0) {
            qg_arrive(&bars->p_full);
            const uint8_t* src = a.image + ((size_t)blockIdx.y * a.jobs + job0) * kSlotBytes;
            int ch = 0;
            for (int c = 0, kr = 0; ch < all_jobs; ch++) {
                // a slot that is handed back has had its copy: the products waited for it
                if (kr && !qg_wait(&bars->x_empty[c], (kr - 1) & 1, bars, a.waits)) break;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc_smem(&bars->x_full[c])), "r"(kSlotBytes)
                             : "memory");
                tc_bulk_g2s(xs + (size_t)c * kSlotBytes, src + (size_t)ch * kSlotBytes, kSlotBytes, &bars->x_full[c]);
                if (++c == a.slots) c = 0, kr++;
            }
            // the last copy of each slot, if nobody else has waited for it
            for (int c = 0; c < min(a.slots, ch); c++)
                for (int it = 0; it < kQgWaits && !qg_try(&bars->x_full[c], (ch - 1 - c) / a.slots & 1); it++) {}
        }
        __syncwarp();
    } else {
        // ---- scales: 0 past the last column's group
        const int t = tid - 18 * 32, groups = (a.w.cols - 1) / a.w.group + 1;   // (a group may be near 2^31)
        uint32_t tile = 0;
        const auto fill = [&](auto* src) {
            using S = typename std::remove_cv<typename std::remove_pointer<decltype(src)>::type>::type;
            constexpr int kPer = 16 / sizeof(S), kDeep = 4;   // scales of a load; loads in flight for each of two rows
            // whole 16-byte loads: the range's first group and the row's last one have to lie on their bounds
            const bool wide = (a.w.lds | groups) % kPer == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0;
            for (int kr = 0; kr < ranges; kr++) {
                const int first = (job0 + kr * a.slots) * 128 / a.w.group;
                for (int b = 0; b < tiles; b++, tile++) {
                    float* to = scales + (tile & 1) * a.groups * 128 + t;
                    const S* p0 = src + min(row0 + b * 128 + t, a.w.rows - 1) * a.w.lds + first;
                    const S* p1 = src + min(row0 + b * 128 + t + 64, a.w.rows - 1) * a.w.lds + first;
                    if (tile > 1 && !qg_wait(&bars->s_empty[tile & 1], (tile >> 1 & 1) ^ 1, bars, a.waits)) return;
                    if (wide && first % kPer == 0) {
                        for (int g0 = 0; g0 < a.groups; g0 += kDeep * kPer) {
                            uint4 u[2][kDeep];
#pragma unroll
                            for (int i = 0; i < kDeep; i++)
                                if (g0 + i * kPer < a.groups && first + g0 + i * kPer < groups) {
                                    u[0][i] = reinterpret_cast<const uint4*>(p0 + g0)[i];
                                    u[1][i] = reinterpret_cast<const uint4*>(p1 + g0)[i];
                                } else {
                                    u[0][i] = u[1][i] = make_uint4(0, 0, 0, 0);
                                }
#pragma unroll
                            for (int i = 0; i < kDeep; i++)
#pragma unroll
                                for (int j = 0; j < kPer; j++)
                                    if (g0 + i * kPer + j < a.groups) {
                                        to[(g0 + i * kPer + j) * 128] = q4_float(reinterpret_cast<const S*>(&u[0][i])[j]);
                                        to[(g0 + i * kPer + j) * 128 + 64] = q4_float(reinterpret_cast<const S*>(&u[1][i])[j]);
                                    }
                        }
                    } else {
#pragma unroll 8
                        for (int g = 0; g < a.groups; g++) {
                            to[g * 128] = first + g < groups ? q4_float(p0[g]) : 0.f;
                            to[g * 128 + 64] = first + g < groups ? q4_float(p1[g]) : 0.f;
                        }
                    }
                    qg_arrive(&bars->s_full[tile & 1]);
                }
            }
        };
        if (a.w.scale_type == FHE_F32) fill(static_cast<const float*>(a.w.scale));
        else if (a.w.scale_type == FHE_F16) fill(static_cast<const __half*>(a.w.scale));
        else fill(static_cast<const __nv_bfloat16*>(a.w.scale));
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (tid == 0 && bars->dead) atomicExch(err, 1u);
    if (warp == 16) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
    }
}

// out = the parts' sum, in their order
template <class T>
__global__ void __launch_bounds__(256) k_q4_sum(const float* __restrict__ parts, int n, int m, int rows, T* __restrict__ out,
                                                long long ldo) {
    pdl_wait();
    const long long each = (long long)m * rows;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < each; i += gridDim.x * 256ll) {
        float v = 0.f;
#pragma unroll 4
        for (int z = 0; z < n; z++) v += parts[z * each + i];
        qg_store(out + i / rows * ldo + i % rows, v);
    }
}
