// Products of two matrices in microscaled 4 bits on the matrix cores: v_mfma_scale_f32_32x32x64_f8f6f4 multiplies 32 x 64 codes by
// 64 x 32 codes under their block scales and adds in fp32.  Lane l of the wave holds row l % 32 and the block l / 32 of an operand:
// exactly one 16-byte block of the row-major form and its scale byte, so operands go from memory to registers as they are.
// 8192^3 in bf16: 257 .. 282 us (3.9 .. 4.3 PFLOP/s), 200 .. 211 with all codes 0, 490 .. 500 at K = 16384.  It takes 474000 cycles whatever the
// codes, of which the matrix pipe is busy 55% (waves wait for 16%); random codes run them at 1.83 GHz, zeros at 2.36: the schedule and the
// chip's power bound it together.  1920 x 12000 x 512 in fp32: 20 us, its 92 MB of y at 4.8 TB/s.  Few tiles (64 x 1024 x 4096: 8.4 us): a
// round trip a stage.
#include "mx4_inl.h"

namespace stattn {

__device__ __forceinline__ i32x8 frag4(uint4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

// Four waves (2 x 2) own a (64 TM) x (64 TN) tile of y, a wave TM x TN tiles of 32 x 32 in its accumulators.  A stage is 256 columns:
// 128 bytes of codes a row, whole cache lines (stages of 128 columns, four in LDS, were 20% slower: a copy's cost is the lines it looks up), and
// its scale bytes.  Two stages in LDS, filled by buffer_load ... lds (no staging registers).
// A fragment read takes chunk 2 ks + (lane / 32) of 32 consecutive rows.  Row r keeps its 16-byte chunk c at position c ^ ((r >> 1) & 7),
// applied to the source address of the copy and to the read: sixteen consecutive lanes then meet sixteen different slots of four banks.
// The pipeline has no gap at a stage's end: the fragments of a step are read while the one before multiplies, the wait for the next
// stage and the barrier stand in front of a stage's last step, whose fragments are in registers by then, and behind that barrier
// nobody reads the stage any more, so the copy of the stage after next starts there.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"     // m0 is written on purpose: it carries the LDS destination of the copy
// 16 bytes a lane from (resource + voff + soff) to LDS byte (lds + 16 * lane); lds and soff are wave-uniform.  Written in asm because
// the compiler would drain every copy in flight in front of the next LDS read; copies are waited for by hand.
__device__ __forceinline__ void copy16(unsigned voff, i32x4v rs, unsigned soff, unsigned lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :: "v"(voff), "s"(rs), "s"(soff), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

// a raw buffer of `bytes`: what lies behind it reads as zero
__device__ __forceinline__ i32x4v buffer_of(const void* p, int64_t bytes) {
    const unsigned long long a = (unsigned long long)p;
    i32x4v rs;
    rs.x = __builtin_amdgcn_readfirstlane((int)(a & 0xffffffffu));
    rs.y = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffffu));
    rs.z = __builtin_amdgcn_readfirstlane((int)(unsigned)min(bytes, (int64_t)0xffffffff));
    rs.w = 0x00020000;
    return rs;
}

template <OpType T, int TM, int TN>
__global__ __launch_bounds__(256) void mx4_gemm_tile_kernel(Mx4GemmArgs p, int tiles_m, int tiles_n) {
    typedef typename Elem<T>::type E;
    constexpr int BM = 64 * TM, BN = 64 * TN, R = BM + BN;
    constexpr int CI = R / 32;                                      // copies of a wave and stage, 8 rows of codes each
    constexpr unsigned STAGE = R * 128u, SCALES = R * 16u;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * STAGE + 2 * SCALES];
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)smem;

    // tiles in order of XCD (block b runs on XCD b % 8), in groups of eight tile rows walked column by column: the 32 tiles an XCD
    // works on at a time are 8 x 4 and share their operands in its L2
    const int nblk = gridDim.x, x = blockIdx.x & 7, q8 = nblk >> 3, r8 = nblk & 7;
    const int lin = x * q8 + min(x, r8) + (blockIdx.x >> 3);
    const int grp = lin / (8 * tiles_n), in = lin - grp * 8 * tiles_n, high = min(8, tiles_m - 8 * grp);
    const int64_t m0 = (int64_t)(8 * grp + in % high) * BM, n0 = (int64_t)(in / high) * BN;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, l31 = lane & 31, g = lane >> 5;
    const int64_t kb = mx4_kp(p.a.cols) / 32;                       // blocks a row
    const unsigned ldc = (unsigned)kb * 16u, lds_ = (unsigned)kb;   // bytes a row of codes, of scales
    const int mlast = (int)min(p.a.rows - m0, (int64_t)BM) - 1, nlast = (int)min(p.w.rows - n0, (int64_t)BN) - 1;
    const i32x4v ra = buffer_of(p.a.codes + m0 * ldc, (p.a.rows - m0) * ldc), rw = buffer_of(p.w.codes + n0 * ldc, (p.w.rows - n0) * ldc);
    const i32x4v rsa = buffer_of(p.a.scales + m0 * lds_, (p.a.rows - m0) * lds_), rsw = buffer_of(p.w.scales + n0 * lds_, (p.w.rows - n0) * lds_);

    // source offsets: a pass of the workgroup copies 32 rows; rows behind the last one repeat it (their results are not stored)
    const int srow = tid >> 3;
    unsigned vo[CI];
#pragma unroll
    for (int i = 0; i < CI; ++i) {
        const int r = 32 * (i < 2 * TM ? i : i - 2 * TM) + srow;
        vo[i] = (unsigned)min(r, i < 2 * TM ? mlast : nlast) * ldc + (unsigned)(((tid & 7) ^ ((r >> 1) & 7)) * 16);
    }
    // scales: 64 rows a wave; a tile with fewer than 256 rows has several waves bring the same ones to the same place
    const int sra = wave * 64 % BM, srw = wave * 64 % BN;
    const unsigned vsa = (unsigned)min(sra + lane, mlast) * lds_, vsw = (unsigned)min(srw + lane, nlast) * lds_;
    const int nsteps = (int)(kb / 2), nstage = (nsteps + 3) / 4;    // steps of 64 columns, stages of four
    constexpr int NC = CI + 1, NF = TM + TN, NP = TM * TN;         // copies, fragments, products of a step
    // Copy number i of what is brought while stage s is finished: the codes of stage s + 2, and one side's scales of 512 columns, 16 bytes
    // a row (a row is a cache line to look up for 16 bytes of scales as for 128 of codes, so they are fetched for two stages at a time):
    // a's from stage s + 3 on where s is odd, w's from stage s + 2 on where it is even.  No branch: the products around it stay in one basic
    // block, where they keep their places.
    auto copy_scales = [&](int q, bool of_a) {
        copy16(of_a ? vsa : vsw, of_a ? rsa : rsw, (unsigned)q * 16u, lds0 + 2 * STAGE + (unsigned)(q & 1) * SCALES + (unsigned)(of_a ? sra : BM + srw) * 16u);
    };
    auto copy_one = [&](int s, int i) {
        if (i < CI) copy16(vo[i], i < 2 * TM ? ra : rw, (unsigned)(s + 2) * 128u, lds0 + (s & 1) * STAGE + (unsigned)wave * 1024u + (unsigned)i * 4096u);
        else copy_scales((s + 3) >> 1, s & 1);
    };

    unsigned fo[4];                                                 // fragment of step ks: row l31 of a 32-row tile
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) fo[ks] = (unsigned)l31 * 128u + (unsigned)(((2 * ks + g) ^ ((l31 >> 1) & 7)) * 16);
    const unsigned sel = 0x06040200u + (unsigned)g * 0x01010101u;   // blocks g, 2 + g, 4 + g, 6 + g of eight
    const unsigned arow = (unsigned)(wm * 32 * TM), wrow = (unsigned)(BM + wn * 32 * TN);

    f32x16v acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    uint4 fa[2][TM], fw[2][TN];
    unsigned sa[TM], sw[TN];                                        // the scale bytes of this lane's blocks in the four steps
    uint2 next[NF];

    auto read_one = [&](int set, int s, int ks, int i) {
        const unsigned char* at = smem + (s & 1) * STAGE + fo[ks];
        const unsigned row = i < TM ? arow + 32u * i : wrow + 32u * (i - TM);
        (i < TM ? fa[set][i] : fw[set][i - TM]) = *reinterpret_cast<const uint4*>(at + row * 128u);
        if (ks == 0) next[i] = *reinterpret_cast<const uint2*>(smem + 2 * STAGE + ((s >> 1) & 1) * SCALES + (s & 1) * 8u + (row + l31) * 16u);
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int i = 0; i < NF; ++i) (i < TM ? sa[i] : sw[i - TM]) = __builtin_amdgcn_perm(next[i].y, next[i].x, sel);
    };
#define MX4_PRODUCT(set, ks, i)                                                                                              \
    acc[(i) / TN][(i) % TN] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(frag4(fa[set][(i) / TN]), frag4(fw[set][(i) % TN]), \
        acc[(i) / TN][(i) % TN], 4, 4, ks, (int)sa[(i) / TN], ks, (int)sw[(i) % TN]);
    // the products of step ks from fragment set `set`; behind each one a share of the next fragments' reads and of the copies, so that
    // the matrix pipe, busy for 32 cycles with a product, covers their issue (the compiler would gather all reads in front)
#define MX4_STEP(ks, READ, next_s, next_ks, COPY, copy_s)                                                                    \
    _Pragma("unroll") for (int i = 0; i < NP; ++i) {                                                                          \
        MX4_PRODUCT((ks) & 1, ks, i)                                                                                               \
        if (READ) { _Pragma("unroll") for (int f = min(2 * i * NF / NP, NF); f < min((2 * i + 2) * NF / NP, NF); ++f) read_one((next_ks) & 1, next_s, next_ks, f); } \
        if (COPY) { _Pragma("unroll") for (int c = i * NC / NP; c < (i + 1) * NC / NP; ++c) copy_one(copy_s, c); }              \
        __builtin_amdgcn_sched_barrier(0);                                                                                   \
    }
#define MX4_ARRIVED(left)                                                                                                        \
    { __builtin_amdgcn_sched_barrier(0); asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(left) : "memory"); __builtin_amdgcn_s_barrier(); __builtin_amdgcn_sched_barrier(0); }
#define MX4_STAGE(s, COPY)                                                                                                   \
    {                                                                                                                        \
        MX4_STEP(0, true, s, 1, false, 0)                                                                                    \
        MX4_STEP(1, true, s, 2, false, 0)                                                                                    \
        MX4_STEP(2, true, s, 3, false, 0)                                                                                    \
        MX4_ARRIVED(0)                                                                                                               \
        MX4_STEP(3, true, (s) + 1, 0, COPY, s)                                                                               \
        take_scales();                                                                                                       \
    }

    copy_scales(0, true);
    for (int s = -2; s < min(0, nstage - 2); ++s) {
#pragma unroll
        for (int i = 0; i < NC; ++i) copy_one(s, i);
    }
    if (nstage > 1) MX4_ARRIVED(NC)
    else MX4_ARRIVED(0)
#pragma unroll
    for (int f = 0; f < NF; ++f) read_one(0, 0, 0, f);
    take_scales();
    int s = 0;
    for (; s + 2 < nstage; ++s) MX4_STAGE(s, true)
    if (s + 1 < nstage) { MX4_STAGE(s, false) ++s; }
    // The last stage has two or four steps (rows are whole multiples of 128 columns).  What stands in LDS for the missing two belongs to
    // other rows: its codes are made 0 and its scales 1, which costs two steps and saves a second copy of the accumulators' code.
    const unsigned keep = 4 * s + 2 < nsteps ? ~0u : 0u;
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = keep ? sa[i] : (sa[i] & 0xffffu) | 0x7f7f0000u;
#pragma unroll
    for (int j = 0; j < TN; ++j) sw[j] = keep ? sw[j] : (sw[j] & 0xffffu) | 0x7f7f0000u;
    auto drop = [&](int set) {
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[set][i] = make_uint4(fa[set][i].x & keep, fa[set][i].y & keep, fa[set][i].z & keep, fa[set][i].w & keep);
    };
    MX4_STEP(0, true, s, 1, false, 0)
    MX4_STEP(1, true, s, 2, false, 0)
    drop(0);
    MX4_STEP(2, true, s, 3, false, 0)
    drop(1);
    MX4_STEP(3, false, 0, 0, false, 0)
#undef MX4_STAGE
#undef MX4_ARRIVED
#undef MX4_STEP
#undef MX4_PRODUCT
    // The products mix lanes, and the compiler moves them freely: the empty statement keeps them in front of the stores' lane-dependent
    // branches, where every lane takes part.
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));

    // Lane: column l31 of each tile, rows 8 (e / 4) + 4 g + e % 4.  Stores go through a buffer that ends behind the last row, lanes behind
    // the last column are sent out of it, so there is no branch; its 32-bit offsets hold because ld_y < 2^22.  Straight stores: through
    // LDS, sixteen bytes a lane, the 8192^3 product took 306 us instead of 290 and the 1920 x 12000 one 26 instead of 20.
    E* y = static_cast<E*>(p.y) + m0 * p.ldy + n0;
    const unsigned ld = (unsigned)p.ldy * (unsigned)sizeof(E);
    const __amdgpu_buffer_rsrc_t ry = __builtin_amdgcn_make_buffer_rsrc(y, 0, (int)((unsigned)(mlast + 1) * ld), 0x00020000);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = wn * 32 * TN + 32 * j + l31;
        const float b = p.bias && n <= nlast ? p.bias[n0 + n] : 0.f;
        const unsigned at = n <= nlast ? (unsigned)(4 * g) * ld + (unsigned)n * (unsigned)sizeof(E) : ~0u;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const E v = (E)(acc[i][j][e] + b);
                const unsigned row = (unsigned)(wm * 32 * TM + 32 * i + 8 * (e >> 2) + (e & 3)) * ld;
                if constexpr (sizeof(E) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), ry, at, row, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), ry, at, row, 0);
            }
    }
}

template <OpType T, int TM, int TN>
static hipError_t run_tiles(hipStream_t s, const Mx4GemmArgs& g) {
    const int64_t tm = (g.a.rows + 64 * TM - 1) / (64 * TM), tn = (g.w.rows + 64 * TN - 1) / (64 * TN);
    mx4_gemm_tile_kernel<T, TM, TN><<<dim3((unsigned)(tm * tn)), 256, 0, s>>>(g, (int)tm, (int)tn);
    return hipGetLastError();
}

// Which tile, measured in bf16 (us): 64 x 64 tiles while all of them run at once, four a CU (300 x 12000 x 512: 5.8, 128 x 128: 6.7;
// 2048 x 2048 x 2048, 1024 tiles: 11.7 against 9.3); 256 x 256 where there are enough of them for half the CUs and the sums are long
// enough to pay for a store that nothing overlaps (13312 x 1024 x 4096: 36 against 42, 3000 x 3000 x 4000, 144 tiles: 32 against 36,
// 4096 x 4096 x 1024: 18.4 against 18.0; 8192 x 8192 x 512: 47 against 40); 128 x 128 otherwise.
template <OpType T>
static hipError_t run(hipStream_t s, const Mx4GemmArgs& g) {
    auto tiles = [&](int64_t edge) { return ((g.a.rows + edge - 1) / edge) * ((g.w.rows + edge - 1) / edge); };
    if (tiles(64) < 4 * 256) return run_tiles<T, 1, 1>(s, g);
    if (tiles(256) >= 128 && g.a.cols > 1024) return run_tiles<T, 4, 4>(s, g);
    return run_tiles<T, 2, 2>(s, g);
}

hipError_t launch_mx4_matmul(hipStream_t s, const Mx4GemmArgs& g) {
    return g.type == OP_F32 ? run<OP_F32>(s, g) : g.type == OP_BF16 ? run<OP_BF16>(s, g) : run<OP_F16>(s, g);
}

}  // namespace stattn
