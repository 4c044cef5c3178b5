// Tile products on the matrix cores: C[m][n] = sum_k A(m,k) B(n,k) over one workgroup's tile.
//
// An operand is either k-contiguous ("KC": element (r,k) at base + r*ld + k) or row-contiguous ("RC": at base + k*ld + r), with rows that
// start on 16 bytes and hold whole 16-byte chunks.  Global reads go through buffer descriptors that start at the tile's corner and end at
// the operand's last element; what lies behind reads as zero, and so do chunks at or behind the contiguous extent, which get an
// offset outside the descriptor.
#pragma once
#include "expert_types.hpp"

namespace ps {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kTileRowBytes = 128;
constexpr unsigned kOutside = 0x80000000u;  // descriptors are kept under 2 GiB

template <typename T>
constexpr int kTileK = kTileRowBytes / (int)sizeof(T);  // k per tile: 32 (fp32), 64 (fp16, bf16)
template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void* base, int64_t bytes) {
  const int n = bytes <= 0 ? 0 : (bytes > 0x7ffffff0 ? 0x7ffffff0 : (int)bytes);
  // (the same in every lane, which the compiler cannot see through the tile search)
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint64_t lo = (unsigned)uniform((int)(unsigned)a), hi = (unsigned)uniform((int)(unsigned)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(lo | (hi << 32)), 0, uniform(n), 0x00027000);
}

// The transposing LDS load.  Without what __restrict__ says here of this one read the compiler takes it to read what the loads under way
// write, and waits for all of them first (the tiles' barriers see to it that they have landed): 65536 rows of 32 experts 2048 x 1024 bf16, input
// gradient 364 us for 306, weights' 304 for 258.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 LdsShorts;
__device__ __forceinline__ u32x2 turned_read(LdsShorts* __restrict__ p) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass drops a kernel's stub over a builtin it does not know)
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
#else
  return u32x2{};
#endif
}

// ------------------------------------------------------------------------------------------------ tiles loaded straight into LDS
// Operands need no registers on the way: buffer loads write LDS directly, 1 KiB per wave and instruction in lane order.  A tile holds 128
// bytes of k and keeps the operand's own direction: KC as rows of k, RC as rows of BR elements of one k each, from which 16-bit fragments
// are read with the transposing LDS loads (16 lanes fetch 4 k x 16 rows, each lane ends up with the 4 k of its row) and fp32 ones element by
// element.  What would collide in the 64 banks is spread by permuting chunks within a tile row, on the global side of the load.
template <typename T, int BR, int NT, bool RC, int KR = kTileK<T>>  // KR: k of an RC tile
struct DirectTile {
  static constexpr int kBytes = RC ? KR * BR * (int)sizeof(T) : BR * kTileRowBytes;
  static constexpr int N = kBytes / 16 / NT;                    // chunks per thread
  static constexpr int kRow = RC ? BR * (int)sizeof(T) : kTileRowBytes;  // bytes of a tile row
  static constexpr int kAcross = kRow / 16;
  static_assert(kBytes % (16 * NT) == 0 && (!RC || kAcross >= 8), "whole chunks per thread; eight chunks to permute among");

  // 16-bit RC: half a wave reads 32 bytes of the eight rows 8 g + (0..3), g = two neighbours; fp32: 64 bytes of four rows 4 g + q
  __device__ static int spread(int row) {
    if constexpr (!RC) {
      return (row >> 1) & 7;
    } else if constexpr (sizeof(T) == 4) {
      return ((row >> 2) & 3) << 2 & (kAcross - 1);
    } else if constexpr (kAcross >= 16) {
      return ((row & 3) | ((row >> 3) & 1) << 2) << 1;
    } else {
      return (((row >> 1) & 1) | ((row >> 3) & 1) << 1) << 1;  // (rows of 128 bytes: their parity is a bank bit already)
    }
  }

  unsigned off[N];  // byte offsets of this thread's chunks from the tile's corner
  int first[N];     // KC: first k, RC: first row of each chunk
  __device__ __forceinline__ void setup(unsigned ld_bytes) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * NT + threadIdx.x, row = id / kAcross, c = (id % kAcross) ^ spread(row);
      off[i] = row * ld_bytes + c * 16;
      first[i] = c * kChunk<T>;
    }
  }
  // left: elements of the contiguous direction from the tile's corner on
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t w, int left, char* lds) const {
    char* base = lds + uniform(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int i = 0; i < N; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (__attribute__((address_space(3))) void*)(base + i * NT * 16), 16, first[i] < left ? off[i] : kOutside, 0,
                                               0, 0);
  }
  // this lane's fragment of the 16 rows from r0 on (a multiple of 16), half s of the tile's k
  __device__ static __forceinline__ u32x4 fragment(const char* lds, int r0, int s) {
    const int r = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    if constexpr (!RC) {
      const int row = r0 + r;
      return *reinterpret_cast<const u32x4*>(lds + row * kTileRowBytes + (((s * 4 + g) ^ spread(r)) << 4));
    } else if constexpr (sizeof(T) == 4) {
      u32x4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = s * 16 + g * 4 + q;
        v[q] = *reinterpret_cast<const unsigned*>(lds + k * kRow + ((((r0 + r) >> 2) ^ spread(k)) << 4) + (r & 3) * 4);
      }
      return v;
    } else {
      u32x4 v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = s * 32 + g * 8 + h * 4 + (r >> 2);
        const char* p = lds + k * kRow + ((((r0 >> 3) + ((r & 3) >> 1)) ^ spread(k)) << 4) + (r & 1) * 8;
        const u32x2 o = turned_read((LdsShorts*)p);
        v[2 * h] = o[0];
        v[2 * h + 1] = o[1];
      }
      return v;
    }
  }
};

// An operand's tiles along k: `rows` rows (KC) or elements of a row (RC) from the tile's corner `base` on, K of k
template <typename T, int BR, int NT, bool RC, int KR = kTileK<T>>
struct DirectSource {
  DirectTile<T, BR, NT, RC, KR> tile;
  const T* base;
  int64_t ld;
  int rows, K;
  __device__ __forceinline__ DirectSource(const T* base_, int64_t ld_, int rows_, int K_) : base(base_), ld(ld_), rows(rows_), K(K_) {
    tile.setup((unsigned)(ld * sizeof(T)));
  }
  __device__ __forceinline__ void load(int k0, char* to) const {
    if constexpr (RC) {
      const int kr = K - k0 < KR ? K - k0 : KR;
      tile.load(window(base + k0 * ld, ((int64_t)(kr - 1) * ld + rows) * sizeof(T)), rows, to);
    } else {
      tile.load(window(base + k0, ((int64_t)(rows - 1) * ld + (K - k0)) * sizeof(T)), K - k0, to);
    }
  }
};

// A barrier behind which all but the last `keep` of every wave's loads have landed in LDS, and every wave has read what it read before.
// (The compiler's own barrier would wait for all of them; it does not know that LDS changes here, hence the empty statements.)
template <int keep>
__device__ __forceinline__ void tile_barrier() {
  static_assert(keep >= 0 && keep < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((keep & 15) | 7 << 4 | 0 << 8 | (keep >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One 16 x 16 block of a product over one fragment of k.  B's rows are the matrix instruction's rows, so a lane ends up with four
// consecutive n of one m: acc[r] = C[lane & 15][4 (lane >> 4) + r].  fp32: the k inside a chunk are taken in the same order for both
// operands, so four 16x16x4 steps consume the four floats of a chunk.
template <typename T>
__device__ __forceinline__ f32x4 mma_block(u32x4 a, u32x4 b, f32x4 acc) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 bf = __builtin_bit_cast(f32x4, b), af = __builtin_bit_cast(f32x4, a);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[q], af[q], acc, 0, 0, 0);
    return acc;
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
  }
}

// ------------------------------------------------------------------------------------------------ which tile where
// Workgroups go round the eight XCDs, each with an L2 of its own.  The tiles of a grid are put in an order in which neighbours share their
// operands' rows -- patches of 32 tiles, what runs on an XCD at a time, up to 8 across -- and the XCDs take patch after patch in turn, the
// last incomplete round in eighths.  (Eighths of the whole order: 343 us where turns take 312, forward, 65536 x 2048 x 1024 bf16, 32 experts.)
constexpr int kXcds = 8, kPatch = 32, kPatchN = 8, kRound = kXcds * kPatch;
inline int64_t xcd_blocks(int64_t tiles) { return (tiles + kXcds - 1) / kXcds * kXcds; }
// the workgroup's place in the order, -1: none
__device__ __forceinline__ int xcd_place(int block, int tiles) {
  const int xcd = block % kXcds, slot = block / kXcds, rounds = tiles / kRound;
  if (slot < rounds * kPatch) return slot / kPatch * kRound + xcd * kPatch + slot % kPatch;
  const int rest = tiles - rounds * kRound, each = (rest + kXcds - 1) / kXcds, in = slot - rounds * kPatch, at = xcd * each + in;
  return in < each && at < rest ? rounds * kRound + at : -1;
}
// the how manieth of the workgroups without a place it is
__device__ __forceinline__ int xcd_spare(int block, int blocks, int tiles) {
  const int rounds = tiles / kRound, rest = tiles - rounds * kRound, each = (rest + kXcds - 1) / kXcds, xcd = block % kXcds;
  auto taken = [&](int x) {
    const int left = rest - x * each;
    return rounds * kPatch + (left < 0 ? 0 : (left < each ? left : each));
  };
  int before = 0;
  for (int x = 0; x < xcd; ++x) before += blocks / kXcds - taken(x);
  return before + block / kXcds - taken(xcd);
}
struct TileAt {
  int m, n;
};
__device__ __forceinline__ TileAt patched_tile(int place, int m_tiles, int n_tiles) {
  const int pn = n_tiles < kPatchN ? n_tiles : kPatchN, pm = kPatch / pn;
  const int band = place / (pm * n_tiles), high = m_tiles - band * pm < pm ? m_tiles - band * pm : pm;
  int in = place - band * pm * n_tiles;
  const int patch = in / (high * pn), wide = n_tiles - patch * pn < pn ? n_tiles - patch * pn : pn;
  in -= patch * high * pn;
  return {band * pm + in / wide, patch * pn + in % wide};
}

}  // namespace ps
