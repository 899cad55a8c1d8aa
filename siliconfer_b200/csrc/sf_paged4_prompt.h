// sf_paged4_prompt.h -- attention over the paged 4-bit cache for long runs of 16-bit queries with 16-bit outputs (part of
// sf_paged4_attention.cu, whose formulas it shares).
//
// A CTA takes 256 query rows of a kv head's group (two tiles of 128, a thread for each row) through all their keys, 128
// at a time, on tcgen05 (kind::f16):
//  * S[row, key] = Q K^T and out[row, d] += P V.  Four warps widen a tile's codes to fp16, a thread for each key: code less
//    8 times the scale of its quarter, relative to a power of two, rounded to 11 bits.  The power is the whole tile's, taken
//    so that its largest element stands at 2^11 to 2^15: a quarter's scale 2^21 below the tile's largest is a normal number
//    still.  A tile whose scales lie further apart is wide: each of its vectors has a power of two of its own, of the scores
//    and of the weights, so that no key's digits hang on another's.  Within a vector, quarters that far below its largest
//    lose digits.  Queries are fp16 numbers after a power of two for the row, weights in fp16.
//  * The sums stay in TMEM; a row that moves its reference multiplies them there.  The tile's powers of two go into the
//    row's factor and reference, so that the softmax has nothing to do for each key but the exponential; a wide tile's keys
//    are multiplied and shifted one by one.
// A key's codes serve 256 rows here and 8 in paged4_attention_kernel.
//
// 8 sequences of 256 tokens with 64 query heads over up to 4000 keys: 214 us, 416 TFLOP/s (paged4_attention_kernel: 887 us);
// 411 us where every tile is wide.
// A tile's keys are widened before the values of the tile before, whose place is free later: the other way round 272 us.
// What is left: items are dealt out whole and in turn, and the SMs work 0.68 of the time there.
#pragma once

constexpr int kPromptRows = 256, kPromptSoft = 8, kPromptThreads = 512, kSlots = 4, kPromptBatch = 2048;
constexpr unsigned kErrProd = 1u << 18, kErrMma = 1u << 19, kErrSoft = 1u << 22, kErrDrain = 1u << 23, kErrWiden = 1u << 24;

constexpr int kHead = 11;         // log2 of the room above a widened element: 8 * 2 * 2^11 is within fp16
constexpr int kSpread = 21;       // exponents that a tile's scales may lie apart: an odd quarter's factor is 2^(11 - 4 - 21) then
constexpr float kFarScore = 0x1p22f;   // above it a score's roundings may pass a weight's room: weights are limited there
constexpr uint32_t kNought = 0x00800000u;   // scales up to 2^-126 are those of zeros

__device__ __forceinline__ uint32_t swizzle128(uint32_t at) { return at ^ ((at >> 3) & 0x70); }

// What the softmax has to know of a tile of keys.
struct TileInfo {
  float k_up;        // of the scores: the keys' power of two
  float v_log;       // log2 of the values' power of two
  float v_down;      // its inverse
  int whole;         // every key of the tile is there
  int wide;          // keys have powers of two of their own
  uint32_t there[4]; // keys that are
  uint32_t nan[4];   // keys whose value is NaN
};

template <int D>
struct Prompt4Lay {
  static constexpr uint32_t ROW = D / 2, T16 = UNIT * D * 2;   // a tile of 128 rows of fp16
  static constexpr uint32_t Q0 = 0, P = UNIT * UNIT * 2, P0 = 2 * T16, K0 = P0 + 2 * P, V0 = K0 + T16;
  static constexpr uint32_t KR = V0 + T16, KS = KR + UNIT * ROW, VS = KS + UNIT * 8, VR = VS + UNIT * 8;
  static constexpr uint32_t CTL = VR + UNIT * ROW, INFO = CTL + 512, POWERS = CTL + 1024, FIRST = POWERS + kSlots * UNIT * 8;
  static constexpr uint32_t TMEM_COLS = 512, O0 = 256;          // scores of two tiles, sums of two tiles
  static constexpr size_t smem(int batch) { return 1024 + FIRST + (size_t)batch * 4; }
  static_assert(sizeof(TileInfo) * kSlots <= 512, "control area");
};

// The 256 rows of a work item, and the keys that some of them see.
struct Prompt4Item {
  int kvh, row0, last_row, r_first, pos0, ta, tb, lo, all_lo, all_hi;   // lo: the first key that some row sees; ta: its tile's
  const int* pages;
};
__device__ __forceinline__ Prompt4Item prompt4_item(const AttnArgs& a, const int* first, int i) {
  int lo = 0;
  for (int hi = a.c.batch; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  const int b = lo, rel = i - first[b];
  Prompt4Item p;
  const int r1 = first_row(a.c, a.T, b + 1);
  p.r_first = first_row(a.c, a.T, b);
  const int n = r1 - p.r_first;
  int len = a.c.seq_lens[b];
  if (!len_ok(a.c, len)) len = 0;
  p.kvh = rel % a.c.n_kv_heads;
  p.row0 = rel / a.c.n_kv_heads * kPromptRows;
  p.last_row = (int)min((long long)p.row0 + kPromptRows, (long long)n * a.G) - 1;
  p.pos0 = len - n;
  p.all_hi = p.pos0 + p.row0 / a.G + 1;
  p.tb = p.pos0 + p.last_row / a.G + 1;
  p.lo = first_seen(a, p.all_hi);
  p.ta = p.lo & ~(UNIT - 1);
  p.all_lo = first_seen(a, p.tb);
  p.pages = a.c.block_table + (size_t)b * a.c.pages_per_seq;
  return p;
}

// Arrives at barrier 2 of the 128 widening threads, and says whether every thread's p is true.
__device__ __forceinline__ int all_of_128(bool p) {
  int all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.and.pred q, 2, 128, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((int)p)
      : "memory");
  return all;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Row `r` of a tile's codes as 16-bit floats, each times its quarter's factor (half2 pairs f; odd quarters' codes are 16
// times as large), in the layout of a K-major or MN-major operand with 128-byte rows of 64 columns.
template <int D>
__device__ __forceinline__ void widen_row(const uint8_t* codes, uint8_t* to, int r, bool live, const uint32_t (&f)[4], uint32_t magic) {
  constexpr int CHUNKS = D / 32, Q = D / 4;   // 16 bytes of codes: 8 places of each quarter
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int chunk = (i + (r >> 1)) & (CHUNKS - 1);   // rows of a phase read from all banks
    uint4 u = *reinterpret_cast<const uint4*>(codes + r * (D / 2) + chunk * 16);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    const auto quarter = [&](auto cc) {
      constexpr int C = decltype(cc)::value;
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = live ? mul_half2(centred<C>(w[j], magic), f[C]) : f[C];
      const int d = C * Q + chunk * 8;
      *reinterpret_cast<uint4*>(to + d / 64 * (UNIT * 128) + swizzle128(r * 128 + d % 64 * 2)) = make_uint4(x[0], x[1], x[2], x[3]);
    };
    quarter(std::integral_constant<int, 0>());
    quarter(std::integral_constant<int, 1>());
    quarter(std::integral_constant<int, 2>());
    quarter(std::integral_constant<int, 3>());
  }
}
// The smallest of four scales that are not those of zeros, less kNought and one bit (more than any number's where all are).
__device__ __forceinline__ uint32_t least_scale(uint2 u) {
  constexpr uint32_t below = kNought + 1;
  return min(min((u.x << 16) - below, (u.x & 0xffff0000u) - below), min((u.y << 16) - below, (u.y & 0xffff0000u) - below));
}
// Factors of a vector's quarters, scale / up with up a power of two, as pairs.
__device__ __forceinline__ void factors(uint2 scales, float down, uint32_t (&f)[4]) {
  float s[4];
  scales_of(scales, s);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float x = s[c] * down * (c % 2 ? 0.0625f : 1.f);
    f[c] = half2_bits(x, x);
  }
}

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1) paged4_prompt_kernel(const __grid_constant__ Attn4Args a, int q_vec) {
  using L = Prompt4Lay<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int wsum[kPromptThreads / 32];
  __shared__ uint32_t tops[2][4][4];   // of a tile, by warp: keys' and values' largest scale, and their smallest
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* mem = smem_raw + (base - raw);
  int* first = reinterpret_cast<int*>(mem + L::FIRST);
  TileInfo* infos = reinterpret_cast<TileInfo*>(mem + L::INFO);
  float2* powers = reinterpret_cast<float2*>(mem + L::POWERS);   // of a wide tile's keys: the key's power, log2 of the value's
  const uint32_t ctl = base + L::CTL;
  const uint32_t krfull = ctl, krempty = ctl + 8, vrfull = ctl + 16, vrempty = ctl + 24, kfull = ctl + 32, kempty = ctl + 40,
                 vfull = ctl + 48, sfull = ctl + 56, sdone = ctl + 72, pfull = ctl + 88, ofull = ctl + 104, qfull = ctl + 120,
                 drain = ctl + 128, ifull = ctl + 136;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(mem + L::CTL + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(mem + L::CTL + 264);
  volatile uint32_t* box_mask = reinterpret_cast<volatile uint32_t*>(mem + L::CTL + 272);   // boxes of a tile that have a page
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    bar_init(krfull, 1);
    bar_init(krempty, 4);
    bar_init(vrfull, 1);
    bar_init(vrempty, 4);
    bar_init(kfull, 4);
    bar_init(kempty, 1);
    bar_init(vfull, 4);
    for (int t = 0; t < 2; ++t) {
      bar_init(sfull + 8 * t, 1);
      bar_init(sdone + 8 * t, 4);
      bar_init(pfull + 8 * t, 4);
      bar_init(ofull + 8 * t, 1);
    }
    bar_init(qfull, kPromptSoft);
    bar_init(drain, 1);
    for (int s = 0; s < kSlots; ++s) bar_init(ifull + 8 * s, 4);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) tmem_alloc(smem_u32((const void*)tmem_slot), L::TMEM_COLS);
  griddep_wait();

  // ---- items before each sequence's ----
  const int B = a.c.batch, Hkv = a.c.n_kv_heads, page_size = a.c.page_size;
  const int rows0 = first_row(a.c, a.T, 0), rows1 = first_row(a.c, a.T, B);
  int total = 0, bad = 0;
  for (int at = 0; at < B; at += kPromptThreads) {
    const int b = at + threadIdx.x;
    int u = 0, off = 0;
    if (b < B) {
      const int r0 = first_row(a.c, a.T, b), r1 = first_row(a.c, a.T, b + 1);
      int n = r1 - r0;
      if (r0 < 0 || n < 0 || r1 > a.T) {
        n = 0;
        off = 1;
        atomicOr(&g_dev_error, kErrIndex);
      }
      if (!len_ok(a.c, a.c.seq_lens[b])) atomicOr(&g_dev_error, kErrIndex);
      u = (int)(((long long)n * a.G + kPromptRows - 1) / kPromptRows) * Hkv;
    }
    int incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < kPromptThreads / 32; ++w) {
      if (w < warp) before += wsum[w];
      total += wsum[w];
    }
    if (b < B) first[b] = before + incl - u;
    bad |= __syncthreads_or(off);
  }
  if (bad) total = 0;
  clear_rows(a, bad ? 0 : rows0, bad ? 0 : rows1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Items in turn, the last rows of a sequence, which see the most keys, first.
  const int items = (int)blockIdx.x < total ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
  const auto item_at = [&](int i) { return prompt4_item(a, first, total - 1 - ((int)blockIdx.x + i * (int)gridDim.x)); };
  const auto tiles_of = [](const Prompt4Item& p) { return p.tb > p.ta ? (p.tb - p.ta + UNIT - 1) / UNIT : 0; };
  const int box = min(page_size, UNIT), boxes = UNIT / box;

  // The launch's 128 registers a thread are dealt out again: 200 * 256 + 40 * 128 + 72 * 128 = 128 * 512.
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---------------- codes to fp16: thread r is key r of a tile ----------------
    // After an expired wait these warps go on through their loops (every wait then returns at once).
    const int r = threadIdx.x - 384, w4 = warp - 12;
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    uint32_t it = 0, vf[4] = {};   // tiles so far; factors of the values of the tile before
    bool v_live = false;
    // the values of tile j
    const auto values = [&](uint32_t j) {
      bar_wait(vrfull, j & 1, kErrWiden, abort_flag);
      if (j > 0) {
        bar_wait(ofull, (j - 1) & 1, kErrWiden, abort_flag);
        bar_wait(ofull + 8, (j - 1) & 1, kErrWiden, abort_flag);
      }
      widen_row<D>(mem + L::VR, mem + L::V0, r, v_live, vf, magic);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        bar_arrive(vfull);
        bar_arrive(vrempty);
      }
    };
    for (int i = 0; i < items; ++i) {
      const Prompt4Item p = item_at(i);
      const int tiles = tiles_of(p);
      for (int k = 0; k < tiles; ++k, ++it) {
        // ---- a tile's keys, then the values of the tile before, whose place is free later ----
        bar_wait(krfull, it & 1, kErrWiden, abort_flag);
        const uint32_t mask = *box_mask;
        const bool there = p.ta + UNIT * k + r < p.tb && (mask >> (r / box) & 1);
        const uint2 none = make_uint2(0, 0);
        const uint2 ks = there ? *reinterpret_cast<const uint2*>(mem + L::KS + 8 * r) : none,
                    vs = there ? *reinterpret_cast<const uint2*>(mem + L::VS + 8 * r) : none;
        const uint32_t kt = __float_as_uint(top_scale(ks)), vt = __float_as_uint(top_scale(vs));
        const bool k_nan = kt >= 0x7f800000u, v_nan = vt >= 0x7f800000u;
        const uint32_t km = __reduce_max_sync(0xffffffffu, k_nan ? 0u : kt), vm = __reduce_max_sync(0xffffffffu, v_nan ? 0u : vt),
                       kl = __reduce_min_sync(0xffffffffu, k_nan ? ~0u : least_scale(ks)),
                       vl = __reduce_min_sync(0xffffffffu, v_nan ? ~0u : least_scale(vs));
        TileInfo& info = infos[it % kSlots];
        const uint32_t have = __ballot_sync(0xffffffffu, there), nans = __ballot_sync(0xffffffffu, v_nan);
        if (lane == 0) {
          tops[it & 1][w4][0] = km;
          tops[it & 1][w4][1] = vm;
          tops[it & 1][w4][2] = kl;
          tops[it & 1][w4][3] = vl;
          info.there[w4] = have;
          info.nan[w4] = nans;
        }
        const int whole = all_of_128(there);
        // exponents, of which a power's inverse is a number, too
        const auto key_power = [](uint32_t top) { return max((int)(top >> 23), kHead + 1); };
        const auto value_power = [](uint32_t top) { return max((int)(top >> 23), 127 - 60); };
        const auto largest = [&](int which) {
          return max(max(tops[it & 1][0][which], tops[it & 1][1][which]), max(tops[it & 1][2][which], tops[it & 1][3][which]));
        };
        const auto far = [&](int which, int power) {   // some scale lies more than kSpread exponents below the power
          const uint32_t x = min(min(tops[it & 1][0][which], tops[it & 1][1][which]), min(tops[it & 1][2][which], tops[it & 1][3][which]));
          return power > kSpread + 1 && x < ((uint32_t)(power - kSpread) << 23) - kNought - 1;
        };
        int ke = key_power(largest(0)), ve = value_power(largest(1));
        const bool wide = far(2, ke) || far(3, ve);
        if (r == 0) {
          info.k_up = __int_as_float((ke - kHead) << 23);
          info.v_log = (float)(ve - kHead - 127);
          info.v_down = __int_as_float((254 + kHead - ve) << 23);
          info.whole = whole;
          info.wide = wide;
        }
        if (wide) {
          ke = key_power(k_nan ? 0u : kt);
          ve = value_power(v_nan ? 0u : vt);
          powers[it % kSlots * UNIT + r] = make_float2(__int_as_float((ke - kHead) << 23), (float)(ve - kHead - 127));
        }
        uint32_t f[4];
        factors(ks, __int_as_float((254 + kHead - ke) << 23), f);
        if (k_nan) f[0] = f[1] = f[2] = f[3] = 0x7e007e00u;
        if (it > 0) bar_wait(kempty, (it - 1) & 1, kErrWiden, abort_flag);
        widen_row<D>(mem + L::KR, mem + L::K0, r, there && !k_nan, f, magic);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          bar_arrive(ifull + 8 * (it % kSlots));
          bar_arrive(kfull);
          bar_arrive(krempty);
        }
        if (it > 0) values(it - 1);
        v_live = there && !v_nan;
        factors(vs, __int_as_float((254 + kHead - ve) << 23), vf);
        if (!v_live) vf[0] = vf[1] = vf[2] = vf[3] = 0u;   // a NaN comes to its rows by their sums
      }
    }
    if (it > 0) values(it - 1);
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 8) {
      // ---------------- copies of codes and scales as they lie ----------------
      uint32_t it = 0;
      bool ok = true;
      const auto bulk = [&](uint32_t dst, const uint8_t* src, uint32_t bytes, uint32_t bar) {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                     "r"(bytes), "r"(bar)
                     : "memory");
      };
      // the values of tile j, asked for after the keys of the next
      uint32_t v_loads = 0;
      const uint8_t* v_from = nullptr;
      const auto values = [&](uint32_t j) {
        if (!__all_sync(0xffffffffu, bar_wait(vrempty, (j & 1) ^ 1, kErrProd, abort_flag))) return false;
        if (lane == 0) bar_expect_tx(vrfull, __popc(v_loads) * (uint32_t)(box * L::ROW));
        __syncwarp();
        if (v_from) bulk(base + L::VR + lane * box * L::ROW, v_from, box * L::ROW, vrfull);
        return true;
      };
      for (int i = 0; i < items && ok; ++i) {
        const Prompt4Item p = item_at(i);
        const auto page_of = [&](int key) {   // a page that ends before the first key may have been given up
          int page = -1;
          if (lane < boxes && key < p.tb && key + box > p.lo) {
            page = __ldg(p.pages + (key >> a.lg_page));
            if ((unsigned)page >= (unsigned)a.c.num_pages) {
              atomicOr(&g_dev_error, kErrIndex);
              page = -1;
            }
          }
          return page;
        };
        int key = p.ta + lane * box, next = page_of(key);
        for (int k0 = p.ta; k0 < p.tb && ok; k0 += UNIT, ++it, key += UNIT) {
          const int page = next;
          next = page_of(key + UNIT);
          const uint32_t loads = __ballot_sync(0xffffffffu, page >= 0);
          const size_t vec = ((size_t)max(page, 0) * Hkv + p.kvh) * page_size + (key & (page_size - 1));
          ok = __all_sync(0xffffffffu, bar_wait(krempty, (it & 1) ^ 1, kErrProd, abort_flag));
          if (!ok) break;
          if (lane == 0) {
            *box_mask = loads;
            bar_expect_tx(krfull, __popc(loads) * (uint32_t)(box * (L::ROW + 16)));
          }
          __syncwarp();
          if (page >= 0) {
            bulk(base + L::KR + lane * box * L::ROW, a.c.k_codes + vec * L::ROW, box * L::ROW, krfull);
            bulk(base + L::KS + lane * box * 8, reinterpret_cast<const uint8_t*>(a.ks) + vec * 8, box * 8, krfull);
            bulk(base + L::VS + lane * box * 8, reinterpret_cast<const uint8_t*>(a.vs) + vec * 8, box * 8, krfull);
          }
          if (it > 0) ok = values(it - 1);
          v_loads = loads;
          v_from = page >= 0 ? a.c.v_codes + vec * L::ROW : nullptr;
        }
      }
      if (ok && it > 0) ok = values(it - 1);
      // every issued copy has landed before the block ends
      if (lane == 0 && ok && it > 0) {
        bar_drain(krfull, (it - 1) & 1, kErrDrain);
        bar_drain(vrfull, (it - 1) & 1, kErrDrain);
      }
      // after an expired wait the copies under way are not counted any more: give them time
      if (!ok) {
        const long long t0 = clock64();
        while (clock64() - t0 < kWaitCycles / 64) {
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---------------- MMAs: the scores of a tile, then the sums of the one before ----------------
      constexpr uint32_t idesc_s = idesc_f16(128, UNIT), idesc_o = idesc_f16(128, D, false, true), h128 = desc_high(1024, kSw128);
      const uint32_t dq = desc_low(base + L::Q0, 16), dk = desc_low(base + L::K0, 16), dp = desc_low(base + L::P0, 16),
                     dv = desc_low(base + L::V0, UNIT * 128);
      uint32_t it = 0, seg = 0;
      bool ok = true;
      const auto scores = [&](uint32_t j) {
        if (!__all_sync(0xffffffffu, bar_wait(kfull, j & 1, kErrMma, abort_flag))) return false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j > 0 && !__all_sync(0xffffffffu, bar_wait(sdone + 8 * t, (j - 1) & 1, kErrMma, abort_flag))) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              mma_f16(tmem + t * UNIT, desc_of(dq + ((t * L::T16 + k / 4 * 16384 + k % 4 * 32) >> 4), h128),
                      desc_of(dk + ((k / 4 * 16384 + k % 4 * 32) >> 4), h128), idesc_s, k != 0);
            mma_commit(sfull + 8 * t);
            if (t == 1) mma_commit(kempty);
          }
          __syncwarp();
        }
        return true;
      };
      const auto sums = [&](uint32_t j, bool begin) {
        if (!__all_sync(0xffffffffu, bar_wait(vfull, j & 1, kErrMma, abort_flag))) return false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!__all_sync(0xffffffffu, bar_wait(pfull + 8 * t, j & 1, kErrMma, abort_flag))) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < UNIT / 16; ++k)
              mma_f16(tmem + L::O0 + t * D, desc_of(dp + ((t * L::P + k / 4 * 16384 + k % 4 * 32) >> 4), h128),
                      desc_of(dv + ((k * 16 * 128) >> 4), h128), idesc_o, !begin || k != 0);
            mma_commit(ofull + 8 * t);
          }
          __syncwarp();
        }
        return true;
      };
      for (int i = 0; i < items && ok; ++i) {
        const int tiles = tiles_of(item_at(i));
        if (tiles == 0) continue;
        ok = __all_sync(0xffffffffu, bar_wait(qfull, seg & 1, kErrMma, abort_flag));
        ++seg;
        if (ok) ok = scores(it);
        for (int k = 0; k < tiles && ok; ++k) {
          if (k + 1 < tiles) ok = scores(it + k + 1);
          if (ok) ok = sums(it + k, k == 0);
        }
        it += tiles;
      }
      // every issued MMA has completed before TMEM is freed
      if (elect_one()) mma_commit(drain);
      __syncwarp();
      bar_drain(drain, 0, kErrDrain);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- softmax: thread tid is row tid of the item ----------------
    // After an expired wait these warps go on through their loops (every wait then returns at once).
    const int tid = threadIdx.x, t = tid >> 7, row_t = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t tmem_s = tmem + lanes + t * UNIT, tmem_o = tmem + lanes + L::O0 + t * D;
    uint32_t it = 0;
    for (int i = 0; i < items; ++i) {
      const Prompt4Item p = item_at(i);
      const int tiles = tiles_of(p);
      const int row = p.row0 + tid, pos = p.pos0 + row / a.G;
      const bool mine = row <= p.last_row;
      float nm = 0.f, l = 0.f;   // minus the reference; the sum
      bool none = true;          // no key yet
      if (tiles > 0) {
        // ---- the row's largest value to [2^13, 2^14) by a power of two; fp16 holds it then as it is ----
        const long long qo = (long long)(p.r_first + row / a.G) * a.qts + (long long)(p.kvh * a.G + row % a.G) * a.qhs;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + qo;
        uint32_t v[D / 2];
        if (q_vec) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = mine ? reinterpret_cast<const uint4*>(q)[c] : make_uint4(0, 0, 0, 0);
            v[4 * c] = w.x, v[4 * c + 1] = w.y, v[4 * c + 2] = w.z, v[4 * c + 3] = w.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < D / 2; ++c) v[c] = mine ? q[2 * c] | (uint32_t)q[2 * c + 1] << 16 : 0u;
        }
        const bool bf16 = a.q_dtype == SF_BF16;
        const auto floats = [&](uint32_t w) {
          return bf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : half2_floats(w);
        };
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < D / 2; ++c) {
          const float2 x = floats(v[c]);
          top = max(top, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
        }
        const int ex = min(max((int)(top >> 23) - 140, -126), 113);
        // a negative scale turns the queries, so that the largest score is the largest sum
        const float down = __int_as_float((127 - ex) << 23) * (a.scale < 0.f ? -1.f : 1.f);
        // an infinity or a NaN: the row is NaN
        const float f = top >= 0x7f800000u ? __int_as_float(0x7fffffff)
                                           : __int_as_float((127 + ex) << 23) * (fabsf(a.scale) * kLog2e);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = floats(v[4 * c + e]);
            w[e] = half2_bits(x.x * down, x.y * down);
          }
          *reinterpret_cast<uint4*>(mem + L::Q0 + t * L::T16 + c / 8 * 16384 + swizzle128(row_t * 128 + c % 8 * 16)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(qfull);

        for (int k = 0; k < tiles; ++k) {
          const uint32_t j = it + k;
          const int k0 = p.ta + UNIT * k;
          bar_wait(sfull + 8 * t, j & 1, kErrSoft, abort_flag);
          __syncwarp();
          tc_fence_after();
          float y[UNIT];
          {
            uint32_t w[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld(tmem_s + 32 * c, w[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_wait(w[c]);
#pragma unroll
              for (int e = 0; e < 32; ++e) y[32 * c + e] = __uint_as_float(w[c][e]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(sdone + 8 * t);
          bar_wait(ifull + 8 * (j % kSlots), (j / kSlots) & 1, kErrSoft, abort_flag);
          const TileInfo& info = infos[j % kSlots];
          float fk = f * info.k_up;
          if (fk < 1e-30f) fk = 1e-30f;   // a hidden key's -inf must stay one; scores this small are none
          const float v_log = info.v_log;
          const bool wide = info.wide;
          const float2* own = powers + j % kSlots * UNIT;
          if (wide || f != f) {   // a NaN row's factor must not meet the -inf of keys that it does not see
#pragma unroll
            for (int e = 0; e < UNIT; ++e) y[e] *= f * own[e].x;
            fk = 1.f;
          }
          // ---- keys that the row does not see ----
          if (!(k0 >= p.all_lo && k0 + UNIT <= p.all_hi && info.whole)) {
            const int hi = max(pos - k0, -1), lo = a.window > 0 ? hi - a.window : -1;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t have = info.there[c];
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * c + e > hi || 32 * c + e <= lo || !(have >> e & 1)) y[32 * c + e] = -INFINITY;
            }
          }
          if (info.nan[0] | info.nan[1] | info.nan[2] | info.nan[3]) {
            const int hi = max(pos - k0, -1), lo = a.window > 0 ? hi - a.window : -1;
            for (int e = 0; e < UNIT; ++e)
              if ((info.nan[e / 32] >> (e % 32) & 1) && e <= hi && e > lo) l = __int_as_float(0x7fffffff);
          }
          // ---- the reference, if a key exceeds it by more than a factor of 2 ----
          float over;
          if (!wide) {
            float m0 = y[0], m1 = y[1], m2 = y[2], m3 = y[3];
#pragma unroll
            for (int e = 4; e < UNIT; e += 4) {
              m0 = fmaxf(m0, y[e]);
              m1 = fmaxf(m1, y[e + 1]);
              m2 = fmaxf(m2, y[e + 2]);
              m3 = fmaxf(m3, y[e + 3]);
            }
            const float most = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
            over = most == -INFINITY ? -INFINITY : most * fk + v_log;
          } else {
            over = -INFINITY;
#pragma unroll
            for (int e = 0; e < UNIT; ++e) over = fmaxf(over, y[e] + own[e].y);
          }
          float c_o = 1.f;
          if (none || over + nm > kTopLog + 1.f) {
            // above what the roundings of a large score may take off, so that its weight is no less than 2^kTopLog
            const float to = fmaf(fabsf(over), 0x1p-22f, kTopLog - over);
            if (none) {
              if (over > -INFINITY) {
                nm = to;
                none = false;
              }
            } else if (!(to >= nm)) {   // an infinite score: NaN
              c_o = ex2(to - nm);
              nm = to;
              l *= c_o;
            }
          }
          // ---- weights, in pairs ----
          uint32_t h[UNIT / 2];
          if (!__any_sync(0xffffffffu, wide || fabsf(nm) > kFarScore)) {
            uint64_t l2 = 0, l3 = 0;   // zeros
            const float base_e = nm + v_log;
            const uint64_t nm2 = pack2(base_e, base_e), fk2 = pack2(fk, fk);
#pragma unroll
            for (int e = 0; e < UNIT; e += 2) {
              float p0, p1;
              unpack2(fma2(pack2(y[e], y[e + 1]), fk2, nm2), p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              if (e & 2) l3 = add2(l3, pack2(p0, p1));
              else l2 = add2(l2, pack2(p0, p1));
              h[e / 2] = half2_bits(p0, p1);
            }
            float l0, l1;
            unpack2(add2(l2, l3), l0, l1);
            l = fmaf(l0 + l1, info.v_down, l);
          } else {
            float ls = 0.f;
#pragma unroll
            for (int e = 0; e < UNIT; e += 2) {
              const float v0 = wide ? own[e].y : v_log, v1 = wide ? own[e + 1].y : v_log;
              const float z0 = at_most(fmaf(y[e], fk, nm), kTopLog + 2.f - v0), z1 = at_most(fmaf(y[e + 1], fk, nm), kTopLog + 2.f - v1);
              ls += ex2(z0) + ex2(z1);
              h[e / 2] = half2_bits(ex2(z0 + v0), ex2(z1 + v1));
            }
            l += ls;
          }
          // ---- the sums of the tile before are there: its P may be written over ----
          if (j > 0) bar_wait(ofull + 8 * t, (j - 1) & 1, kErrSoft, abort_flag);
          __syncwarp();
          tc_fence_after();
          if (__any_sync(0xffffffffu, c_o != 1.f)) {   // by whole warps, as TMEM is read and written
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t w[32];
              tmem_ld(tmem_o + c, w);
              tmem_wait(w);
#pragma unroll
              for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * c_o);
              tmem_st(tmem_o + c, w);
            }
            tmem_wait_st();
          }
#pragma unroll
          for (int c = 0; c < UNIT / 8; ++c)
            *reinterpret_cast<uint4*>(mem + L::P0 + t * L::P + c / 8 * 16384 + swizzle128(row_t * 128 + c % 8 * 16)) =
                make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
          fence_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(pfull + 8 * t);
        }
        it += tiles;
        bar_wait(ofull + 8 * t, (it - 1) & 1, kErrSoft, abort_flag);
        __syncwarp();
        tc_fence_after();
      }
      // ---- the row's result ----
      const size_t th = (size_t)(p.r_first + row / a.G) * a.H + p.kvh * a.G + row % a.G;
      const float g = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t w[16] = {};
        __syncwarp();
        if (tiles > 0) {
          tmem_ld(tmem_o + c, w);
          tmem_wait(w);
        }
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = l == 0.f ? 0.f : __uint_as_float(w[e]) * g;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          if (!mine) break;
          const float z[8] = {x[e], x[e + 1], x[e + 2], x[e + 3], x[e + 4], x[e + 5], x[e + 6], x[e + 7]};
          if (a.out_dtype == SF_F16) store8(static_cast<__half*>(a.out) + th * D + c + e, z);
          else store8(static_cast<__nv_bfloat16*>(a.out) + th * D + c + e, z);
        }
      }
      tc_fence_before();   // the next item's sums overwrite these columns after this warp's arrival at pfull
      if (mine && a.lse) a.lse[th] = l == 0.f ? -INFINITY : -nm * kLn2 + logf(l);
    }
  }
  griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_free(tmem, L::TMEM_COLS);
  }
}

template <int D>
int launch_prompt4(const Attn4Args& a, long long items, bool q_vec, cudaStream_t st) {
  using L = Prompt4Lay<D>;
  auto* fn = paged4_prompt_kernel<D>;
  static_assert(L::smem(kPromptBatch) + 512 <= kBlockSmem, "shared memory plan");
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem(kPromptBatch));
  if (e != cudaSuccess) return cuda_fail(e, "paged4_prompt_kernel shared memory");
  const int sms = device_info().sms;
  e = launch_kernel(fn, items < sms ? (int)items : sms, kPromptThreads, L::smem(a.c.batch), st, true, a, (int)q_vec);
  if (e != cudaSuccess) return cuda_fail(e, "paged4_prompt_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}
