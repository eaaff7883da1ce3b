// Which of its forms a dense product (vm_linear) takes, and its grid: on the host, without HIP.
#pragma once

#include <stdint.h>

namespace vm {

// Rows up to which a block reads its matrix rows once for all of them, without MFMA: eight rows 7.6 us by 2560 x 2560,
// in 16 x 16 tiles 6.8; four 5.8.
constexpr uint32_t kFewRows = 4;
constexpr int kFewMatrix = 4;             // matrix rows of a block there
constexpr uint32_t kFewWaves = 8;         // waves at most, each over every so manyth kilobyte of the rows

// Tiles of a form: their rows and matrix rows, a block's threads, how many of them a CU holds at once, and the us in which it
// computes one alone and all that it holds: a fixed part and one per 32 inputs.  Fitted by hand to calls of 512 to 2560 inputs
// and one to six rounds of tiles in either format (an MX step of 64 inputs takes about what two of bf16 take); for other
// sizes it is an extrapolation, which chooses among forms that are all right for them.
struct TileForm {
  uint32_t rows, matrix, threads, places;
  float one, one_step, full, full_step;
};
enum : int { kForm16, kForm32, kForm32x64, kForm64, kForm64Deep, kForm128, kForm128x320, kForm256, kForm256x320, kForms };
enum : int { kFormFew = -1 };
constexpr uint32_t kCus = 256;
template <bool MX>
inline constexpr TileForm kTileForms[kForms] = {
    {16, 16, 512, 2, 2.5f, 0.045f, 2.5f, 0.060f},        // 8 waves, each every eighth chunk
    {32, 32, 1024, 2, 3.5f, 0.058f, 4.0f, 0.090f},       // 16 waves, each every fourth
    {32, 64, 512, 2, 3.5f, 0.080f, 5.0f, 0.100f},        // 8 waves, each every other
    {64, 64, 256, 3, 6.0f, 0.100f, 8.0f, 0.220f},        // 4 waves
    {64, 64, 512, 1, 5.5f, 0.075f, 5.5f, 0.075f},        // 8 waves, each every other chunk
    {128, 128, 512, 2, 5.9f, 0.277f, 9.0f, 0.500f},      // the large tiles of two groups of waves
    {128, 320, 512, 1, 14.0f, 0.450f, 14.0f, 0.450f},
    {256, 256, 512, 1, 12.0f, 0.580f, 12.0f, 0.580f},
    {256, 320, 512, 1, 18.0f, 0.820f, 18.0f, 0.820f},
};
template <>
inline constexpr TileForm kTileForms<true>[kForms] = {
    {16, 16, 512, 2, 2.5f, 0.042f, 2.5f, 0.050f},
    {32, 32, 1024, 2, 3.5f, 0.058f, 4.0f, 0.080f},
    {32, 64, 512, 3, 3.8f, 0.085f, 6.0f, 0.165f},
    {64, 64, 256, 3, 5.0f, 0.137f, 8.0f, 0.235f},
    {64, 64, 512, 0, 0.0f, 0.000f, 0.0f, 0.000f},        // no faster than 32 x 64: not built
    {128, 128, 512, 2, 5.9f, 0.240f, 9.0f, 0.400f},
    {128, 320, 512, 1, 14.0f, 0.450f, 14.0f, 0.450f},
};

// A call's form, its blocks and their threads, and whether no CU holds two of its tiles.
struct LinearForm {
  int form;
  uint64_t blocks;
  uint32_t threads;
  bool alone;
  // a grid's threads are counted in 32 bits
  bool fits() const { return (blocks * threads >> 32) == 0; }
};

// `n` outputs of a row, two matrix rows each with `pairs` (SwiGLU); `large`: rows lie near enough for the large tiles, and MX
// scales move as words.  The form of the least time by the model.
template <bool MX>
inline LinearForm choose_form(uint32_t rows, uint32_t n, uint32_t k_bytes, bool pairs, bool large) {
  const uint64_t matrix = pairs ? uint64_t(n) * 2 : n;
  if (rows <= kFewRows) {
    const uint32_t kilobytes = (k_bytes + 1023) / 1024;
    return {kFormFew, (matrix + kFewMatrix - 1) / kFewMatrix, 64 * (kilobytes < kFewWaves ? kilobytes : kFewWaves), false};
  }
  const float steps = static_cast<float>(k_bytes) / (MX ? 32.0f : 64.0f);
  // of MX 256 x 320 would outgrow the LDS, and 256 x 256 is slower than 128 x 320 (a full round of the chip 62 us for 52, of a
  // fifth fewer products)
  const int forms = large ? (MX ? kForm256 : kForms) : kForm128;
  LinearForm best{kForm16, 0, 0, false};
  float least = 0.0f;
  for (int f = 0; f < forms; ++f) {
    const TileForm& t = kTileForms<MX>[f];
    if (t.places == 0) continue;
    const uint64_t tiles = uint64_t((rows + t.rows - 1) / t.rows) * ((matrix + t.matrix - 1) / t.matrix);
    const uint64_t left = tiles % (t.places * kCus), held = (left + kCus - 1) / kCus;   // by a CU, of the last round
    const float one = t.one + t.one_step * steps, full = t.full + t.full_step * steps;
    float us = static_cast<float>(tiles / (t.places * kCus)) * full;
    if (held > 0) us += t.places == 1 ? full : one + (full - one) * static_cast<float>(held - 1) / static_cast<float>(t.places - 1);
    if (best.blocks == 0 || us < least) {
      least = us;
      best = {f, tiles, t.threads, tiles <= kCus};
    }
  }
  return best;
}

}  // namespace vm
