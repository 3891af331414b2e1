// Matrix product of 8-bit integers with a scale a row (token, pixel) and a scale a channel:
//   y[m][n] = act( (sum_k a[m][k] * w[n][k]) * (a_scale[m] * w_scale[n]) + bias[n] )
// The sum is exact: products of 8-bit integers in 32-bit accumulators, at most Y5_I8_MAX_K of them.  One rounding to the output type.
#include "y5_common.h"

namespace {

#include "conv_common.h"

#include "gemm_i8.h"

// ------------------------------------------------------------------------------------------ phased kernel
// The schedule of conv_ph.hip on bytes: eight waves as WM x WN, each owning MF x NF accumulators of v_mfma_i32_16x16x64_i8; a
// K-tile is 128 bytes of every row, staged as four half-tiles (row halves P0 / P1 = the waves' first / second MF halves, channel
// halves W0 / W1) into a ring of four slots by buffer_load ... lds, up to 1.5 K-tiles ahead; two phases a K-tile, waves 4-7 one
// barrier behind waves 0-3, so that on every SIMD one wave multiplies while its partner reads LDS and issues copies; the only
// wait for copies is a counted s_waitcnt vmcnt(N) that leaves the youngest half-tiles in flight.  128-byte LDS rows are
// XOR-swizzled through the copies' source addresses.  Rows and bytes past the matrices fail the descriptors' range check and
// arrive as zeros; descriptors start at the tile, so the matrices may be of any size.
// Measured: 16384 x 4096 x 4096 in 209 us alone (2.63 POP/s; 214 behind its quantisation), the 8-bit library product of the same sizes
// 267.  Bound by the clock that the matrix units' load leaves: a K-tile of 256 x 256 takes 1.4 us with every unit busy, its matrix
// instructions alone 0.85 at 2.4 GHz.  12800 x 1024 x 512: 13 us, one round of 200 tiles whose eight K-tiles take 7 of them.
// Hazards.  RAW: a half-tile is read no earlier than the phase after the counted wait that retired it, behind a barrier every
// wave has passed after its own wait.  WAR: a slot is refilled one phase after its last read, and every phase drains its reads
// (lgkmcnt(0)) before its first barrier.
template <int WM, int WN, int MF, int NF>
struct GemmCfg {
    static_assert(WM * WN == 8 && MF >= 2 && NF >= 2 && MF * NF <= 32, "eight waves, at most 128 accumulator registers");
    static constexpr int MF0 = (MF + 1) / 2, MF1 = MF / 2, NF0 = (NF + 1) / 2, NF1 = NF / 2;
    static constexpr int BM = WM * MF * 16, BN = WN * NF * 16;
    static_assert(BM <= 512 && BN <= 512, "one scale a thread");
    static constexpr int PR = MF0 * 16, WR = NF0 * 16;                    // rows a wave row / wave column owns in a slot
    static constexpr int P_SLOT = WM * PR * 128, W_SLOT = WN * WR * 128;  // bytes
    static constexpr int P_PIECES = WM * PR / 8, W_PIECES = WN * WR / 8;  // 1 KiB copies of a half-tile
    static constexpr int NP = (P_PIECES + 7) / 8, NW = (W_PIECES + 7) / 8;
    static constexpr bool DUMP = (P_PIECES % 8) != 0 || (W_PIECES % 8) != 0;  // some waves issue a piece past the slot:
    static constexpr int RING = 4 * (P_SLOT + W_SLOT);                        // it zero-fills 1 KiB behind the rings
    static constexpr int PRM_AT = RING + (DUMP ? 1024 : 0);  // scales of the rows, scales and biases of the channels
    static constexpr int SMEM = PRM_AT + (BM + 2 * BN) * 4;
    static_assert(SMEM <= 160 * 1024, "one workgroup per compute unit");
};

// The copy as in conv_ph.hip: M0 is left at its LDS address
__device__ __forceinline__ void dma16_m0(i32x4 rsrc, unsigned voff, unsigned lds_base) {
    asm volatile(
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen lds"
        :
        : "v"(voff), "s"(rsrc), "s"(lds_base)
        : "memory", "m0");
}

#define GP_SYNC_READS() asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory")
#define GP_BARRIER() asm volatile("s_barrier" ::: "memory")

template <typename T, int ACT, int WM, int WN, int MF, int NF>
__global__ __launch_bounds__(512, 2) void gemm_ph_kernel(const GemmArgs g) {
    typedef GemmCfg<WM, WN, MF, NF> Cfg;
    constexpr int MF0 = Cfg::MF0, MF1 = Cfg::MF1, NF0 = Cfg::NF0, NF1 = Cfg::NF1;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, PR = Cfg::PR, WR = Cfg::WR;
    constexpr int P_SLOT = Cfg::P_SLOT, W_SLOT = Cfg::W_SLOT, W_RING = 4 * P_SLOT;
    constexpr int NP = Cfg::NP, NW = Cfg::NW;
    constexpr int VM = 2 * NP + 2 * NW;  // four half-tiles (P1, P0, W0, W1) stay in flight at the wait of a phase
    constexpr int CH = 4 * NF;           // consecutive channels of a lane
    constexpr int SV = 16 / (int)sizeof(T), ST = MF * CH / SV;  // values of a store, stores of a tile
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];

    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int late = wave >> 2;
    const int nk = g.nk, ld = g.ld;
    // lane l of a 1 KiB copy fills 16-byte slot (l & 7) of row (l >> 3), which holds chunk (l & 7) ^ f(row), f(row) = (row >> 1) & 7
    const int kc = (lane & 7) ^ (((wave & 1) << 2) | (lane >> 4));
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)smem;
    const int lr = lane & 15, lq = lane >> 4;
    const int sw = (lr >> 1) & 7;
    int coff[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) coff[ks] = ((4 * ks + lq) ^ sw) << 4;
    const unsigned char* prow = smem + (wm * PR + lr) * 128;
    const unsigned char* wrow = smem + W_RING + (wn * WR + lr) * 128;
    float* prm = reinterpret_cast<float*>(smem + Cfg::PRM_AT);

    // Byte offsets of this lane's chunk 0 in the rows it copies; the same for every tile.  Row `within` of a half-tile's wave column
    // is the channel that gives a lane consecutive ones: accumulator j, element e of lane (lr, lq) is channel lq * CH + 4 j + e.
    unsigned pbase[2][NP], wbase[2][NW];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = wave + 8 * i, r = p * 8 + (lane >> 3);
            const int wv = r / PR, within = r - wv * PR;
            const bool valid = p < Cfg::P_PIECES && within < (h ? MF1 : MF0) * 16;
            pbase[h][i] = valid ? (unsigned)((wv * (MF * 16) + h * (MF0 * 16) + within) * ld + kc * 16) : Y5_BUF_OOB;
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int p = wave + 8 * i, r = p * 8 + (lane >> 3);
            const int wv = r / WR, within = r - wv * WR;
            const bool valid = p < Cfg::W_PIECES && within < (h ? NF1 : NF0) * 16;
            const int j = h * NF0 + (within >> 4), q = within & 15;
            wbase[h][i] = valid ? (unsigned)((wv * (NF * 16) + (q >> 2) * CH + 4 * j + (q & 3)) * ld + kc * 16) : Y5_BUF_OOB;
        }
    }
    // the offset of K-tile kt; past a row's end (or the last K-tile) one that fails the range check: a tile's rows span less than
    // 2^30 bytes
    auto koff = [&](int kt) -> unsigned { return kt * 128 + kc * 16 < ld ? (unsigned)kt * 128u : 0x40000000u; };
    auto issue_p = [&](const i32x4& pr, int h, int slot, unsigned ko) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const bool out = 8 * i + 7 >= Cfg::P_PIECES && wave + 8 * i >= Cfg::P_PIECES;
            const unsigned dst = out ? (unsigned)Cfg::RING : (unsigned)(slot * P_SLOT + (wave + 8 * i) * 1024);
            dma16_m0(pr, pbase[h][i] + ko, lds0 + dst);
        }
    };
    auto issue_w = [&](const i32x4& wr, int h, int slot, unsigned ko) {
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const bool out = 8 * i + 7 >= Cfg::W_PIECES && wave + 8 * i >= Cfg::W_PIECES;
            const unsigned dst = out ? (unsigned)Cfg::RING : (unsigned)(W_RING + slot * W_SLOT + (wave + 8 * i) * 1024);
            dma16_m0(wr, wbase[h][i] + ko, lds0 + dst);
        }
    };

    struct Tile {
        long long m0;
        int n0, rows_m, rows_n;
        float as, ws, b;  // this thread's row and channel
    } cur;
    i32x4 pr, wr;
    unsigned ko;
    // a tile's place, its scales, and the copies of K-tile 0 and of P0, W0, W1 of K-tile 1, in the order the loop continues
    auto start = [&](int it) {
        const int tile = xcd_remap(it, g.tiles_total);
        const int mt = tile / g.tiles_n, nt = tile - mt * g.tiles_n;
        cur.m0 = (long long)mt * BM;
        cur.n0 = nt * BN;
        cur.rows_m = g.m - cur.m0 < BM ? (int)(g.m - cur.m0) : BM;
        cur.rows_n = g.n - cur.n0 < BN ? g.n - cur.n0 : BN;
        pr = make_buf(g.a + cur.m0 * ld, cur.rows_m * ld);
        wr = make_buf(g.w + (long long)cur.n0 * ld, cur.rows_n * ld);
        cur.as = t < cur.rows_m ? g.a_scale[cur.m0 + t] : 0.f;
        cur.ws = t < cur.rows_n ? g.w_scale[cur.n0 + t] : 0.f;
        cur.b = t < cur.rows_n && g.bias ? g.bias[cur.n0 + t] : 0.f;
        ko = koff(0);
        issue_p(pr, 0, 0, ko);
        issue_w(wr, 0, 0, ko);
        issue_w(wr, 1, 1, ko);
        issue_p(pr, 1, 1, ko);
        ko = koff(1);
        issue_p(pr, 0, 2, ko);
        issue_w(wr, 0, 2, ko);
        issue_w(wr, 1, 3, ko);
    };

    i32x4 pf[MF0][2], wf[NF][2], acc[MF][NF];
#define GP_READ_P(SLOT, N)                                                                           \
    _Pragma("unroll") for (int i = 0; i < (N); ++i)                                                  \
        _Pragma("unroll") for (int ks = 0; ks < 2; ++ks)                                             \
            pf[i][ks] = *reinterpret_cast<const i32x4*>(prow + (SLOT) * P_SLOT + i * 2048 + coff[ks]);
#define GP_READ_W(J0, SLOT, N)                                                                       \
    _Pragma("unroll") for (int j = 0; j < (N); ++j)                                                  \
        _Pragma("unroll") for (int ks = 0; ks < 2; ++ks)                                             \
            wf[(J0) + j][ks] = *reinterpret_cast<const i32x4*>(wrow + (SLOT) * W_SLOT + j * 2048 + coff[ks]);
#define GP_MMA(M0, MN)                                                                               \
    __builtin_amdgcn_sched_barrier(0);                                                               \
    __builtin_amdgcn_s_setprio(1);                                                                   \
    _Pragma("unroll") for (int ks = 0; ks < 2; ++ks)                                                 \
        _Pragma("unroll") for (int i = 0; i < (MN); ++i)                                             \
            _Pragma("unroll") for (int j = 0; j < NF; ++j)                                           \
                acc[(M0) + i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j][ks], pf[i][ks], acc[(M0) + i][j], 0, 0, 0); \
    __builtin_amdgcn_s_setprio(0);                                                                   \
    __builtin_amdgcn_sched_barrier(0);

    start(blockIdx.x);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(NP + 2 * NW) : "memory");  // K-tile 0 has landed for every wave
    for (int it = blockIdx.x; it < g.tiles_total; it += gridDim.x) {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
        if (late) GP_BARRIER();
        for (int kt = 0; kt < nk; ++kt) {
            const int s0 = (2 * kt) & 3, s1 = s0 + 1;
            // phase A: rows P0 x channels W0 | W1; P1 of K-tile kt+1 goes where P1 of kt-1 was
            GP_READ_P(s0, MF0)
            GP_READ_W(0, s0, NF0)
            GP_READ_W(NF0, s1, NF1)
            issue_p(pr, 1, (s1 + 2) & 3, ko);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VM) : "memory");
            GP_SYNC_READS();
            GP_MMA(0, MF0)
            GP_BARRIER();
            // phase B: rows P1, the weights still in registers; P0, W0, W1 of K-tile kt+2 go where this K-tile's were
            GP_READ_P(s1, MF1)
            ko = koff(kt + 2);
            issue_p(pr, 0, s0, ko);
            issue_w(wr, 0, s0, ko);
            issue_w(wr, 1, s1, ko);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(VM) : "memory");
            GP_SYNC_READS();
            GP_MMA(MF0, MF1)
            GP_BARRIER();
        }
        if (!late) GP_BARRIER();
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");  // the zero fills of the last K-tiles are in: the ring is free

        if (t < BM) prm[t] = cur.as;
        if (t < BN) {
            prm[BM + t] = cur.ws;
            prm[BM + BN + t] = cur.b;
        }
        // the next tile's first copies fly while this one's results are scaled and stored, straight from the registers
        const Tile done = cur;
        const bool more = it + (int)gridDim.x < g.tiles_total;
        if (more) start(it + (int)gridDim.x);
        GP_SYNC_READS();
        // accumulator (i, j): row wm*MF*16 + i*16 + lr; element e is channel wn*NF*16 + lq*CH + 4*j + e
        const int nl = wn * (NF * 16) + lq * CH;
        T* yt = static_cast<T*>(g.y) + done.m0 * g.y_ld + done.n0;
        const BufRsrc yr = make_rsrc(yt, (int)(((long long)(done.rows_m - 1) * g.y_ld + done.rows_n) * (int)sizeof(T)));
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            int ml = wm * (MF * 16) + i * 16 + lr;
            asm volatile("" : "+v"(ml));  // its addresses are made here, not kept for MF rows through the K loop
            const float as = prm[ml];
            T out[CH];
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const f32x4 ws = *reinterpret_cast<const f32x4*>(prm + BM + nl + 4 * j), bs = *reinterpret_cast<const f32x4*>(prm + BM + BN + nl + 4 * j);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][e] * (as * ws[e]) + bs[e];
                act_n<ACT>(v, g.slope);
#pragma unroll
                for (int e = 0; e < 4; ++e) out[4 * j + e] = (T)v[e];
            }
            if (g.whole) {  // every row starts on 16 bytes and the channels are whole vectors: ST stores a wave, whatever the tile
#pragma unroll
                for (int k = 0; k < CH / SV; ++k) {
                    typedef T Vec __attribute__((ext_vector_type(SV)));
                    Vec o;
#pragma unroll
                    for (int e = 0; e < SV; ++e) o[e] = out[k * SV + e];
                    const unsigned off = ml < done.rows_m && nl + k * SV < done.rows_n ? (unsigned)(ml * (int)g.y_ld + nl + k * SV) * (unsigned)sizeof(T) : Y5_BUF_OOB;
                    st16_buf(__builtin_bit_cast(i32x4, o), yr, off);
                }
            } else if (ml < done.rows_m) {
#pragma unroll
                for (int k = 0; k < CH / SV; ++k) {
                    T* p = yt + ml * g.y_ld + nl + k * SV;
                    if (nl + (k + 1) * SV <= done.rows_n) {
                        st_out<T, SV>(p, out + k * SV);
                    } else {
#pragma unroll
                        for (int e = 0; e < SV; ++e)
                            if (nl + k * SV + e < done.rows_n) p[e] = out[k * SV + e];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // one row's values at a time: the accumulators leave no room for more
        }
        if (!more) break;
        // K-tile 0 of the next tile has landed for every wave: all but the copies behind it and the ST stores behind those (where
        // their number is not known, the stores are waited for too)
        if (g.whole) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NP + 2 * NW + ST < 63 ? NP + 2 * NW + ST : 63) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        GP_SYNC_READS();
    }
}
#undef GP_READ_P
#undef GP_READ_W
#undef GP_MMA

template <typename T, int ACT, int WM, int WN, int MF, int NF>
int launch_ph(GemmArgs g, hipStream_t st) {
    typedef GemmCfg<WM, WN, MF, NF> Cfg;
    g.nk = (g.ld + 127) / 128;
    g.whole = y5_aligned16(g.y) && g.y_ld * (long long)sizeof(T) % 16 == 0 && g.n * (int)sizeof(T) % 16 == 0 && g.y_ld * (long long)sizeof(T) * Cfg::BM < 0x40000000LL;
    g.tiles_n = (g.n + Cfg::BN - 1) / Cfg::BN;
    const long long total = (g.m + Cfg::BM - 1) / Cfg::BM * g.tiles_n;
    Y5_REQUIRE(total <= 0x7fffffffLL, "gemm_i8: %lld tiles", total);
    g.tiles_total = (int)total;
    static std::atomic<unsigned long long> attr_set{0};  // one bit per device: the attribute is per function and device
    const unsigned long long bit = 1ull << y5_current_device();
    if (!(attr_set.load() & bit)) {
        Y5_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_ph_kernel<T, ACT, WM, WN, MF, NF>), hipFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        attr_set.fetch_or(bit);
    }
    const long long cus = cu_count();
    const unsigned grid = (unsigned)(total < cus ? total : cus);
    hipLaunchKernelGGL((gemm_ph_kernel<T, ACT, WM, WN, MF, NF>), dim3(grid), dim3(512), Cfg::SMEM, st, g);
    Y5_LAUNCH_CHECK("gemm_ph_kernel");
    return Y5_OK;
}

// The phased tiles, and what a launch of one costs (us): a round of tiles over the chip takes `round` + `ktile` for each K-tile, both
// measured with every compute unit busy (16384 x 4096 x 4096: 209 / 253 / 353 / 519 us in the order below; 12800 x 1024 x 512: 18.2 /
// 13.2 / 16.3 / 23.7; 2048 x 2048 x 2048: 24.9 / 17.7 / 15.2 / 21.0; 1000 x 1000 x 1000: 19.7 / 12.7 / 9.6 / 8.1 - the model is within 15 % of
// each).  A large tile reads LDS less often for each product, a small one leaves fewer units idle in the last round.
struct PhTile {
    int bm, bn;
    float round, ktile;
};
constexpr PhTile kPhTiles[] = {{256, 256, 6.5f, 1.4f}, {256, 128, 3.5f, 0.85f}, {128, 128, 2.5f, 0.6f}, {128, 64, 2.f, 0.45f}};
constexpr float kPhLaunch = 2.f;

float ph_cost(const GemmArgs& g, const PhTile& p) {
    const long long tiles = (g.m + p.bm - 1) / p.bm * ((g.n + p.bn - 1) / p.bn), cus = cu_count();
    return kPhLaunch + (float)((tiles + cus - 1) / cus) * (p.round + p.ktile * (float)((g.ld + 127) / 128));
}

int best_ph(const GemmArgs& g) {
    int best = 0;
    for (int i = 1; i < 4; ++i)
        if (ph_cost(g, kPhTiles[i]) < ph_cost(g, kPhTiles[best])) best = i;
    return best;
}

// The kernel for little work (gemm_i8_few.hip) with rows x 16 outputs a workgroup: a launch, the workgroups' starts, what they read
// through the caches at 10 TB/s, the weights from memory at 5 (us; measured 64 x 1024 x 1024: 3.3 / 4.1 for 16 / 32 rows, 400 x 512 x
// 512: 4.4, 16 x 4096 x 4096: 6.6, 64 x 4096 x 4096: 17.1 / 13.7, 256 x 1024 x 1024: 6.5 / 5.5 - phased: 6.8, 5.1, 17.9, 17.7, 6.9)
float few_cost(const GemmArgs& g, int rows) {
    const float wgs = (float)((g.m + rows - 1) / rows) * (float)((g.n + 15) / 16);
    return (rows == 16 ? 2.2f : 2.8f) + 1e-3f * wgs + 1e-7f * wgs * (float)(rows + 16) * (float)g.ld + 2e-7f * (float)g.n * (float)g.ld;
}

template <typename T, int ACT>
int gemm(const GemmArgs& g, hipStream_t st) {
    switch (best_ph(g)) {
        case 0: return launch_ph<T, ACT, 2, 4, 8, 4>(g, st);
        case 1: return launch_ph<T, ACT, 4, 2, 4, 4>(g, st);
        case 2: return launch_ph<T, ACT, 4, 2, 2, 4>(g, st);
        default: return launch_ph<T, ACT, 4, 2, 2, 2>(g, st);
    }
}

template <typename T>
int gemm_act(const GemmArgs& g, hipStream_t st) {
    if (g.act == Y5_ACT_LEAKY) return gemm<T, Y5_ACT_LEAKY>(g, st);
    if (g.act == Y5_ACT_SILU) return gemm<T, Y5_ACT_SILU>(g, st);
    return gemm<T, Y5_ACT_NONE>(g, st);
}

int check(const y5_gemm_i8_desc& d) {
    Y5_REQUIRE(d.w && d.w_scale && d.y, "gemm_i8: null tensor pointer");
    Y5_REQUIRE(d.dtype == Y5_F16 || d.dtype == Y5_BF16 || d.dtype == Y5_F32, "gemm_i8: dtype %d", d.dtype);
    Y5_REQUIRE(d.m > 0 && d.m <= 0x7fffffff && d.n > 0 && d.n <= 1 << 20, "gemm_i8: %lld rows, %d channels", (long long)d.m, d.n);
    Y5_REQUIRE(d.k > 0 && d.k <= Y5_I8_MAX_K, "gemm_i8: %d values a row (1 to %d)", d.k, Y5_I8_MAX_K);
    Y5_REQUIRE(d.ld == (d.k + 15) / 16 * 16, "gemm_i8: a row of a and w is %d bytes for %d values (got %d)", (d.k + 15) / 16 * 16, d.k, d.ld);
    Y5_REQUIRE(d.y_ld >= d.n, "gemm_i8: output pitch %lld for %d channels", (long long)d.y_ld, d.n);
    Y5_REQUIRE(d.act == Y5_ACT_NONE || d.act == Y5_ACT_LEAKY || d.act == Y5_ACT_SILU, "gemm_i8: activation %d", d.act);
    Y5_REQUIRE((y5_aligned16(d.a) && y5_aligned16(d.w)), "gemm_i8: a and w must be 16-byte aligned");
    const int es = d.dtype == Y5_F32 ? 4 : 2;
    Y5_REQUIRE(reinterpret_cast<uintptr_t>(d.y) % es == 0 && reinterpret_cast<uintptr_t>(d.a_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(d.w_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(d.bias) % 4 == 0, "gemm_i8: misaligned pointer");
    return Y5_OK;
}

}  // namespace

int y5_launch_gemm_i8(const y5_gemm_i8_desc& d, hipStream_t st) {
    Y5_REQUIRE(d.a && d.a_scale, "gemm_i8: null tensor pointer");
    if (int rc = check(d)) return rc;
    // Many rows of few values: the weights fit LDS and the tiles' fixed costs outweigh their reuse (819200 x 64 x 64: 29 us against 53 of
    // the best tile, 204800 x 256 x 64: 17 against 24, 204800 x 256 x 256: 37 against 40, 204800 x 512 x 128: 35 against 36, 51200 x 64 x
    // 64: 4.6 against 6.4; but 51200 x 128 x 128: 7.4 against 7.6, 51200 x 512 x 128: 14 against 11, 12800 x 256 x 256: 8.8 against 5.8)
    if (y5_gemm_rows_fits(d.n, d.k, false, d.dtype) && (d.m >= 65536 || (d.k <= 64 && d.m >= 4096))) return y5_launch_gemm_rows(d, nullptr, 0, st);
    const GemmArgs g = make_gemm_args(d);
    const float few = few_cost(g, 16), few2 = few_cost(g, 32);
    if (d.m <= 1 << 20 && (few < few2 ? few : few2) < ph_cost(g, kPhTiles[best_ph(g)])) return y5_launch_gemm_few(d, nullptr, 0, few < few2 ? 16 : 32, st);
    if (d.dtype == Y5_F16) return gemm_act<f16>(g, st);
    if (d.dtype == Y5_BF16) return gemm_act<bf16>(g, st);
    return gemm_act<float>(g, st);
}

namespace {
// Whether linear_i8 quantises inside the product: a few rows by every workgroup, or many rows of few values in the registers that
// read them
enum { kTwoSteps, kFew, kRows };
int fused(const y5_gemm_i8_desc& d, int x_dtype) {
    if (x_dtype != d.dtype) return kTwoSteps;
    // 1 x 4096 x 4096: 6.3 us in one, 10.9 in two; 4 x 4096 x 4096: 8.7 and 11.5; every workgroup quantises all rows, so not more
    if (d.m <= Y5_FEW_ROWS && d.m * d.ld <= 64 * 1024) return kFew;
    // The one launch has the weights to lay out in every workgroup's LDS before its rows (4096 x 128 x 128: 5.3 us in one, 6.5 in two; 819200
    // x 64 x 64: 39 and 55; 204800 x 256 x 256: 46 and 65; 12800 x 512 x 64: 9.1 and 13.1; but 12800 x 256 x 256: 10.7 and 10.8, 16384 x
    // 512 x 256: 18.1 and 16.3, 2048 x 64 x 64 in fp32: 5.9 and 5.3)
    return d.m >= 4096 && d.m >= (int64_t)d.n * d.k / 4 && y5_gemm_rows_fits(d.n, d.k, true, d.dtype) ? kRows : kTwoSteps;
}
}  // namespace

int y5_linear_i8_work(const y5_gemm_i8_desc& d, int x_dtype, size_t* bytes) {
    *bytes = fused(d, x_dtype) ? 0 : (size_t)d.m * d.ld + (size_t)d.m * sizeof(float);
    return Y5_OK;
}

int y5_launch_linear_i8(const y5_gemm_i8_desc& d0, const void* x, int64_t x_ld, int x_dtype, void* workspace, size_t workspace_bytes, hipStream_t st) {
    y5_gemm_i8_desc d = d0;
    d.a = d.a_scale = nullptr;
    if (int rc = check(d)) return rc;
    Y5_REQUIRE(x, "linear_i8: null x");
    Y5_REQUIRE(x_dtype == Y5_F16 || x_dtype == Y5_BF16 || x_dtype == Y5_F32, "linear_i8: x dtype %d", x_dtype);
    Y5_REQUIRE(x_ld >= d.k, "linear_i8: pitch %lld for %d values", (long long)x_ld, d.k);
    Y5_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == Y5_F32 ? 4 : 2) == 0, "linear_i8: misaligned x");
    const int how = fused(d, x_dtype);
    if (how == kFew) return y5_launch_gemm_few(d, x, x_ld, 16, st);
    if (how == kRows) return y5_launch_gemm_rows(d, x, x_ld, st);
    size_t need = 0;
    if (int rc = y5_linear_i8_work(d, x_dtype, &need)) return rc;
    if (!workspace || workspace_bytes < need) return y5_fail(Y5_EWORKSPACE, "linear_i8: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
    Y5_REQUIRE(y5_aligned16(workspace), "linear_i8: misaligned workspace");
    float* scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + (size_t)d.m * d.ld);
    if (int rc = y5_launch_quantize_rows(x, x_ld, x_dtype, d.m, d.k, workspace, d.ld, scale, st)) return rc;
    d.a = workspace;
    d.a_scale = scale;
    return y5_launch_gemm_i8(d, st);
}
