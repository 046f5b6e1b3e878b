// The threads that hold a row in registers, in chunks of eight elements: host code of its own, so that plans made of it can be asked without a GPU.
#pragma once

namespace cf {

constexpr int kRowWave = 64;
// threads of a row, V chunks each
constexpr int row_threads(int H, int V) { return ((H + 7) / 8 + kRowWave * V - 1) / (kRowWave * V) * kRowWave; }
constexpr int kOneWaveH = 8 * kRowWave, kOneChunkH = 8 * 1024;

}  // namespace cf
