// sf_paged_prompt.h -- attention over the paged e4m3 cache for long runs of bf16 queries with 16-bit outputs (part of
// sf_paged_attention.cu, whose formulas, reference and query scaling it shares).
//
// A CTA takes 256 query rows of a kv head's group (two tiles of 128, a thread for each row) through all their keys, 128
// at a time:
//  * S[row, key] = Q K^T on the cache's codes (kind::f8f6f4), a row's two parts added in the accumulator: the nearest
//    e4m3 numbers, and what these lack in e5m2.  That is at most 8 last places of a bf16 number, which 3 bits hold, so
//    it is exact; elements below 2^-14 of the row's largest lose what lies under 2^-21 of that.
//  * out[row, d] += P V (kind::f16): weights in fp16, 2^-11 of each and no coarser than 2^-37 of the reference; V's
//    codes, which are fp16 numbers, are widened by the softmax warps.  Its sums stay in TMEM; a row that moves its
//    reference multiplies them there.
// Two parts in fp8 or one in fp16 cost the tensor cores the same; fp16 weights take one conversion where two e4m3 parts
// take seven instructions, and widening V costs a thread 64 codes for its 128 keys.
//
// A key's bytes serve 256 rows here and 8 in paged_attention_kernel.  8 sequences of 256 tokens with 64 query heads over
// up to 4000 keys: 197 us, 451 TFLOP/s (paged_attention_kernel: 700 us); a tile of 128 keys takes 3.2 us, of which the
// tensor cores work 1.1.
#pragma once

constexpr int kPromptRows = 256, kPromptSoft = 8, kPromptThreads = 384, kSlots = 4;
// A launch of 384 threads has 168 registers each, a row's thread needs more: 224 * 256 + 56 * 128 = 168 * 384.
constexpr float kPromptScale = 8192.f;   // of a weight: at most 2^14, within fp16

template <int D>
struct PromptLay {
  static constexpr int INNER = D;                            // 64 or 128 bytes a row: one sub-tile
  static constexpr uint32_t TILE = UNIT * D;
  static constexpr uint32_t Q = 128 * D, P = 128 * 256, V16 = UNIT * D * 2;
  static constexpr uint32_t Q0 = 0, P0 = Q0 + 4 * Q, K0 = P0 + 2 * P, V0 = K0 + 2 * TILE, W0 = V0 + TILE;
  static constexpr uint32_t CTL = W0 + V16, SCALES = CTL + 512, FIRST = CTL + 1024;
  static constexpr uint64_t SWZ = INNER == 128 ? kSw128 : kSw64;
  static constexpr uint32_t TMEM_COLS = 512, O0 = 256;       // scores of two tiles, sums of two tiles
  static constexpr size_t smem(int batch) { return 1024 + FIRST + (size_t)batch * 4; }
};

__device__ __forceinline__ uint32_t swizzle(uint32_t at, int inner) { return at ^ ((at >> 3) & (inner == 128 ? 0x70 : 0x30)); }

// The 256 rows of a work item, and the keys that some of them see.
struct PromptItem {
  int kvh, row0, last_row, r_first, pos0, ta, tb, lo, all_lo, all_hi;   // lo: the first key that some row sees; ta: its tile's
  const int* pages;
};
__device__ __forceinline__ PromptItem prompt_item(const AttnArgs& a, const int* first, int i) {
  int lo = 0;
  for (int hi = a.c.batch; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  const int b = lo, rel = i - first[b];
  PromptItem p;
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

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                        const AttnArgs a, int q_vec) {
  using L = PromptLay<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int wsum[kPromptThreads / 32];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* mem = smem_raw + (base - raw);
  int* first = reinterpret_cast<int*>(mem + L::FIRST);
  const uint32_t ctl = base + L::CTL;
  const uint32_t kfull = ctl, kempty = ctl + 16, vfull = ctl + 32, vempty = ctl + 40, sfull = ctl + 48, sdone = ctl + 64,
                 pfull = ctl + 80, ofull = ctl + 88, qfull = ctl + 96, drain = ctl + 104, cfull = ctl + 112;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(mem + L::CTL + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(mem + L::CTL + 264);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      bar_init(kfull + 8 * s, 1);
      bar_init(kempty + 8 * s, 1);
      bar_init(sfull + 8 * s, 1);
      bar_init(sdone + 8 * s, 4);
    }
    bar_init(vfull, 1);
    bar_init(vempty, kPromptSoft);
    bar_init(pfull, kPromptSoft);
    bar_init(ofull, 1);
    bar_init(qfull, kPromptSoft);
    bar_init(drain, 1);
    for (int s = 0; s < kSlots; ++s) bar_init(cfull + 8 * s, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 && lane == 0) {
    prefetch_map(&mapK);
    prefetch_map(&mapV);
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
  const auto item_at = [&](int i) { return prompt_item(a, first, total - 1 - ((int)blockIdx.x + i * (int)gridDim.x)); };

  if (warp >= kPromptSoft) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");   // one instruction for the warpgroup
  if (warp == 8) {
    // ---------------- page copies; a tile's scales to its slot ----------------
    const int box = min(page_size, UNIT), boxes = UNIT / box;
    uint32_t it = 0, nv = 0, v_bytes = 0;
    int v_y = 0;
    bool ok = true, v_load = false;
    const auto values = [&] {
      if (!__all_sync(0xffffffffu, bar_wait(vempty, (nv & 1) ^ 1, kErrProd, abort_flag))) return false;
      if (lane == 0) bar_expect_tx(vfull, v_bytes);
      __syncwarp();
      if (v_load) tma_load(base + L::V0 + lane * box * L::INNER, &mapV, 0, v_y, vfull);
      ++nv;
      return true;
    };
    for (int i = 0; i < items && ok; ++i) {
      const PromptItem p = item_at(i);
      // lane l: page of box l two tiles ahead, its scales one tile ahead
      constexpr long long kNoKey = 1ll << 32;   // no page number, right or wrong
      const auto page_of = [&](int key) -> long long {   // a page that ends before the first key may have been given up
        return lane < boxes && key < p.tb && key + box > p.lo ? __ldg(p.pages + (key >> a.lg_page)) : kNoKey;
      };
      struct Box {
        int page;
        float ks, vs;
      };
      const auto scales_of = [&](long long page) {
        Box x{-1, 0.f, 0.f};
        if (page >= 0 && page < a.c.num_pages) {
          x.page = (int)page;
          x.ks = __ldg(a.c.k_scales + (size_t)page * Hkv + p.kvh);
          x.vs = __ldg(a.c.v_scales + (size_t)page * Hkv + p.kvh);
        } else if (page != kNoKey) {
          atomicOr(&g_dev_error, kErrIndex);
        }
        return x;
      };
      int key = p.ta + lane * box;
      Box nxt = scales_of(page_of(key));
      long long page2 = page_of(key + UNIT);
      for (int k0 = p.ta; k0 < p.tb && ok; k0 += UNIT, ++it, key += UNIT) {
        const Box cur = nxt;
        nxt = scales_of(page2);
        page2 = page_of(key + 2 * UNIT);
        const bool load = cur.page >= 0;
        const int y = load ? (cur.page * Hkv + p.kvh) * page_size + (key & (page_size - 1)) : 0;
        const int loads = __popc(__ballot_sync(0xffffffffu, load));
        const uint32_t bytes = loads * (uint32_t)(box * D);
        const bool all = loads == boxes;
        const uint32_t s = it & 1;
        ok = __all_sync(0xffffffffu, bar_wait(kempty + 8 * s, ((it >> 1) & 1) ^ 1, kErrProd, abort_flag));
        if (!ok) break;
        if (lane < boxes)
          *reinterpret_cast<float4*>(mem + L::SCALES + (it % kSlots) * 128 + lane * 16) =
              make_float4(cur.ks, cur.vs * kPromptScale, fmaxf(lg2(cur.vs), -60.f), all ? 2.f : load ? 1.f : 0.f);
        __syncwarp();
        if (lane == 0) {
          bar_arrive(cfull + 8 * (it % kSlots));
          bar_expect_tx(kfull + 8 * s, bytes);
        }
        __syncwarp();
        if (load) tma_load(base + L::K0 + s * L::TILE + lane * box * L::INNER, &mapK, 0, y, kfull + 8 * s);
        if (it > 0) ok = values();   // the next tile's K is asked for before this one's V has to be free
        v_load = load;
        v_y = y;
        v_bytes = bytes;
      }
    }
    if (ok && it > 0) ok = values();
    // every issued copy has landed before the block ends
    if (lane == 0 && ok) {
      for (uint32_t j = it < 2 ? 0 : it - 2; j < it; ++j) bar_drain(kfull + 8 * (j & 1), (j >> 1) & 1, kErrDrain);
      if (nv > 0) bar_drain(vfull, (nv - 1) & 1, kErrDrain);
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
    constexpr uint32_t idesc_s = idesc_e4m3(128, UNIT), idesc_r = idesc_s | kAE5m2, idesc_o = idesc_f16(128, D, false, true);
    constexpr uint32_t hk = desc_high(8 * L::INNER, L::SWZ), h128 = desc_high(1024, kSw128);
    const uint32_t dk = desc_low(base + L::K0, 16), dq = desc_low(base + L::Q0, 16), dp = desc_low(base + L::P0, 16),
                   dw = desc_low(base + L::W0, UNIT * 128);
    uint32_t it = 0;
    bool ok = true;
    const auto scores = [&](uint32_t j) {
      const uint32_t s = j & 1;
      if (!__all_sync(0xffffffffu, bar_wait(kfull + 8 * s, (j >> 1) & 1, kErrMma, abort_flag))) return false;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (j > 0 && !__all_sync(0xffffffffu, bar_wait(sdone + 8 * t, (j - 1) & 1, kErrMma, abort_flag))) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t k0 = dk + s * (L::TILE >> 4);
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
              mma_f8(tmem + t * UNIT, desc_of(dq + (((2 * t + part) * L::Q + k * 32) >> 4), hk), desc_of(k0 + k * 2, hk),
                     part ? idesc_r : idesc_s, part + k != 0);
          mma_commit(sfull + 8 * t);
          if (t == 1) mma_commit(kempty + 8 * s);
        }
        __syncwarp();
      }
      return true;
    };
    const auto sums = [&](uint32_t j) {
      if (!__all_sync(0xffffffffu, bar_wait(pfull, j & 1, kErrMma, abort_flag))) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < UNIT / 16; ++k)
            mma_f16(tmem + L::O0 + t * D, desc_of(dp + ((t * L::P + k / 4 * 16384 + k % 4 * 32) >> 4), h128),
                    desc_of(dw + ((k * 16 * 128) >> 4), h128), idesc_o, 1);
        mma_commit(ofull);
      }
      __syncwarp();
      return true;
    };
    uint32_t seg = 0;
    for (int i = 0; i < items && ok; ++i) {
      const PromptItem p = item_at(i);
      const int tiles = p.tb > p.ta ? (p.tb - p.ta + UNIT - 1) / UNIT : 0;
      if (tiles == 0) continue;
      ok = __all_sync(0xffffffffu, bar_wait(qfull, seg & 1, kErrMma, abort_flag));
      ++seg;
      if (ok) ok = scores(it);
      for (int k = 0; k < tiles && ok; ++k) {
        if (k + 1 < tiles) ok = scores(it + k + 1);
        if (ok) ok = sums(it + k);
      }
      it += tiles;
    }
    // every issued MMA has completed before TMEM is freed
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    bar_drain(drain, 0, kErrDrain);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ---------------- softmax: thread tid is row tid of the item ----------------
    // After an expired wait these warps go on through their loops (every wait then returns at once).
    const int tid = threadIdx.x, t = tid >> 7, row_t = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t tmem_s = tmem + lanes + t * UNIT, tmem_o = tmem + lanes + L::O0 + t * D;
    const int lg_box = min(a.lg_page, 7);
    uint32_t it = 0;
    for (int i = 0; i < items; ++i) {
      const PromptItem p = item_at(i);
      const int tiles = p.tb > p.ta ? (p.tb - p.ta + UNIT - 1) / UNIT : 0;
      const int row = p.row0 + tid, pos = p.pos0 + row / a.G;
      const bool mine = row <= p.last_row;
      float nm = 0.f, l = 0.f;   // minus the reference; the sum
      bool fresh = true;         // no key yet
      if (tiles > 0) {
        // ---- the row's two parts; the sums' zeros ----
        const long long qo = (long long)(p.r_first + row / a.G) * a.qts + (long long)(p.kvh * a.G + row % a.G) * a.qhs;
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + qo;
        uint32_t v[D / 2];
        uint32_t top = 0;
        if (q_vec) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = mine ? reinterpret_cast<const uint4*>(q)[c] : make_uint4(0, 0, 0, 0);
            v[4 * c] = w.x, v[4 * c + 1] = w.y, v[4 * c + 2] = w.z, v[4 * c + 3] = w.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < D / 2; ++c) {
            const unsigned short* s = reinterpret_cast<const unsigned short*>(q) + 2 * c;
            v[c] = mine ? s[0] | (uint32_t)s[1] << 16 : 0u;
          }
        }
#pragma unroll
        for (int c = 0; c < D / 2; ++c) top = max(top, max(v[c] << 16 & 0x7fff0000u, v[c] & 0x7fff0000u));
        // the row's largest value to [128, 256) by a power of two; an infinity would saturate: its row is NaN
        const int ex = min(max((int)(top >> 23) - 134, -126), 126);
        const float down = __int_as_float((127 - ex) << 23);
        const float f = top >= 0x7f800000u ? __int_as_float(0x7fffffff)
                                           : __int_as_float((127 + ex) << 23) * (a.scale * kLog2e);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t w0[4], w1[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = v[8 * c + 2 * e], y = v[8 * c + 2 * e + 1];
            float z[4] = {__uint_as_float(x << 16) * down, __uint_as_float(x & 0xffff0000u) * down,
                          __uint_as_float(y << 16) * down, __uint_as_float(y & 0xffff0000u) * down};
            w0[e] = take_e4m3(z);   // leaves 16 times what they lack
            w1[e] = to_e5m2x2(z[0] * 0.0625f, z[1] * 0.0625f) | to_e5m2x2(z[2] * 0.0625f, z[3] * 0.0625f) << 16;
          }
          const uint32_t at = swizzle(row_t * L::INNER + c * 16, L::INNER);
          *reinterpret_cast<uint4*>(mem + L::Q0 + 2 * t * L::Q + at) = make_uint4(w0[0], w0[1], w0[2], w0[3]);
          *reinterpret_cast<uint4*>(mem + L::Q0 + (2 * t + 1) * L::Q + at) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
        }
        {
          uint32_t z[16] = {};
#pragma unroll
          for (int c = 0; c < D; c += 16) tmem_st(tmem_o + c, z);
          tmem_wait_st();
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
          bar_wait(cfull + 8 * (j % kSlots), (j / kSlots) & 1, kErrSoft, abort_flag);
          const float4* scales = reinterpret_cast<const float4*>(mem + L::SCALES + (j % kSlots) * 128);
          const bool whole = k0 >= p.all_lo && k0 + UNIT <= p.all_hi;   // every row sees all of these keys
          // ---- scores; the reference, if a key exceeds it by more than a factor of 2 ----
          float over = -INFINITY;
          if (whole && scales[0].w == 2.f) {
#pragma unroll
            for (int c = 0; c < UNIT / 16; ++c) {
              const float4 sc = scales[c * 16 >> lg_box];
              const float fk = f * sc.x;
              const uint64_t fk2 = pack2(fk, fk);
              float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
              for (int e = 16 * c; e < 16 * c + 16; e += 2) {
                unpack2(mul2(pack2(y[e], y[e + 1]), fk2), y[e], y[e + 1]);
                m0 = fmaxf(m0, y[e]);
                m1 = fmaxf(m1, y[e + 1]);
              }
              over = fmaxf(over, fmaxf(m0, m1) + sc.z);
            }
          } else {
            const int hi = max(pos - k0, -1), lo = a.window > 0 ? hi - a.window : -1;
#pragma unroll
            for (int c = 0; c < UNIT / 16; ++c) {
              const float4 sc = scales[c * 16 >> lg_box];
              const float fk = f * sc.x;
              const int to = sc.w == 0.f ? -1 : hi;
              float m = -INFINITY;
#pragma unroll
              for (int e = 16 * c; e < 16 * c + 16; ++e) {
                y[e] = e > to || e <= lo ? -INFINITY : y[e] * fk;
                m = fmaxf(m, y[e]);
              }
              over = fmaxf(over, m + sc.z);
            }
          }
          float c_o = 1.f;
          if (fresh) {
            if (over > -INFINITY) {
              nm = -over;
              fresh = false;
            }
          } else if (over + nm > 1.f) {
            c_o = ex2(-(over + nm));
            nm = -over;
            l *= c_o;
          }
          // ---- weights, in pairs ----
          uint32_t h[UNIT / 2];
          uint64_t l2 = 0;   // two zeros
          const uint64_t nm2 = pack2(nm, nm);
#pragma unroll
          for (int c = 0; c < UNIT / 16; ++c) {
            const float fold = scales[c * 16 >> lg_box].y;
            const uint64_t fold2 = pack2(fold, fold);
#pragma unroll
            for (int e = 16 * c; e < 16 * c + 16; e += 2) {
              float p0, p1;
              unpack2(add2(pack2(y[e], y[e + 1]), nm2), p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              const uint64_t pp = pack2(p0, p1);
              l2 = add2(l2, pp);
              unpack2(mul2(pp, fold2), p0, p1);
              const __half2 x = __floats2half2_rn(p0, p1);
              h[e / 2] = *reinterpret_cast<const uint32_t*>(&x);
            }
          }
          {
            float l0, l1;
            unpack2(l2, l0, l1);
            l += l0 + l1;
          }
          // ---- the sums of the tile before are there: its P and V may be written over ----
          if (j > 0) bar_wait(ofull, (j - 1) & 1, kErrSoft, abort_flag);
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
            *reinterpret_cast<uint4*>(mem + L::P0 + t * L::P + c / 8 * 16384 + swizzle(row_t * 128 + c % 8 * 16, 128)) =
                make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
          // ---- V to fp16: key row_t, this half of the head's columns ----
          bar_wait(vfull, j & 1, kErrSoft, abort_flag);
          {
            const bool seen = k0 + row_t < p.tb && scales[row_t >> lg_box].w != 0.f;   // else 0, whatever lies there
            uint32_t nan = 0;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              const int d = t * (D / 2) + 16 * c;
              uint4 u = *reinterpret_cast<const uint4*>(mem + L::V0 + swizzle(row_t * L::INNER + d, L::INNER));
              if (!seen) u = make_uint4(0, 0, 0, 0);
              const uint32_t in[4] = {u.x, u.y, u.z, u.w};
              uint32_t out[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t x = in[e];
                const uint32_t bad = ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                // where not all rows see the key, a NaN code is 0 here and comes to its rows below
                if (!whole && bad) {
                  nan = 1;
                  x &= ~(bad | (bad - (bad >> 7)));
                }
                const __half2_raw a0 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x & 0xffffu), __NV_E4M3),
                                  a1 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x >> 16), __NV_E4M3);
                out[2 * e] = (uint32_t)a0.x | (uint32_t)a0.y << 16;
                out[2 * e + 1] = (uint32_t)a1.x | (uint32_t)a1.y << 16;
              }
              uint8_t* w = mem + L::W0 + d / 64 * (UNIT * 128);
              *reinterpret_cast<uint4*>(w + swizzle(row_t * 128 + d % 64 * 2, 128)) = make_uint4(out[0], out[1], out[2], out[3]);
              *reinterpret_cast<uint4*>(w + swizzle(row_t * 128 + d % 64 * 2 + 16, 128)) = make_uint4(out[4], out[5], out[6], out[7]);
            }
            if (!whole && any_of<256>(nan != 0)) {
              for (int kk = 0; kk < UNIT && k0 + kk < p.tb; ++kk) {
                if (scales[kk >> lg_box].w == 0.f) continue;
                const bool sees = k0 + kk <= pos && (a.window <= 0 || k0 + kk > pos - a.window);
                for (int d = 0; d < D; ++d) {
                  if ((mem[L::V0 + swizzle(kk * L::INNER + d, L::INNER)] & 0x7fu) != 0x7fu) continue;
                  uint32_t w;
                  __syncwarp();
                  tmem_ld1(tmem_o + d, w);
                  if (sees) w = 0x7fffffffu;
                  tmem_st1(tmem_o + d, w);
                  tmem_wait_st();
                }
              }
            }
          }
          fence_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            bar_arrive(vempty);
            bar_arrive(pfull);
          }
        }
        it += tiles;
        bar_wait(ofull, (it - 1) & 1, kErrSoft, abort_flag);
        tc_fence_after();
      }
      // ---- the row's result ----
      const size_t th = (size_t)(p.r_first + row / a.G) * a.H + p.kvh * a.G + row % a.G;
      const float g = l == 0.f ? 0.f : 1.f / (l * kPromptScale);
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
int launch_prompt(const AttnArgs& a, long long items, bool q_vec, cudaStream_t st) {
  using L = PromptLay<D>;
  const sf_paged_cache& c = a.c;
  const uint64_t rows = (uint64_t)c.num_pages * c.n_kv_heads * c.page_size;
  if (rows > 0x7fffffffull) return fail(SF_ERR_UNSUPPORTED, "the cache has more than 2^31 - 1 rows");
  const CUtensorMapSwizzle swz = L::INNER == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const uint32_t box = c.page_size < UNIT ? c.page_size : UNIT;
  CUtensorMap mk, mv;
  if (!make_tensor_map(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.k_codes, D, rows, D, L::INNER, box, swz) ||
      !make_tensor_map(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.v_codes, D, rows, D, L::INNER, box, swz))
    return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled failed for the cache");
  auto* fn = paged_prompt_kernel<D>;
  const size_t smem = L::smem(c.batch);
  static_assert(L::smem(kMaxBatch) + 1024 <= kBlockSmem, "shared memory plan");
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem(kMaxBatch));
  if (e != cudaSuccess) return cuda_fail(e, "paged_prompt_kernel shared memory");
  const int sms = device_info().sms;
  e = launch_kernel(fn, items < sms ? (int)items : sms, kPromptThreads, smem, st, true, mk, mv, a, (int)q_vec);
  if (e != cudaSuccess) return cuda_fail(e, "paged_prompt_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}
