// tg_attn_split.h — how tg_attention_shared cuts its work: host arithmetic
// alone, without a device or CUDA's headers.
#pragma once
#include <algorithm>
#include <cmath>

namespace tg {

constexpr int AT_ROWS = 128;    // query rows per tile (MMA M)
constexpr int AT_KEYS = 128;    // keys per block (MMA N of S, K of P V)
constexpr int OWN_KEYS = 128;   // own keys per stage: 32 for each warp of a group

struct SharedSplit {
  int tpt, units;     // tokens of a tile; units (pairs of tiles) of the batch
  int gp, nt, ngc;    // query heads of a key head, rounded up to 8; groups of 8 of them at a time; such turns
  int nsp = 0;        // pieces of the prefix
  int own_ctas = 0;   // SMs of the own keys
  SharedSplit(int B, int P, int max_len, int H, int KH, int hd, int sms) {
    const int G = H / KH, HD = hd <= 64 ? 64 : 128;
    tpt = AT_ROWS / G;
    units = (B + 2 * tpt - 1) / (2 * tpt);
    nt = G <= 8 ? 1 : 2;
    ngc = (G + 8 * nt - 1) / (8 * nt);
    gp = (G + 7) / 8 * 8;
    if (B == 0) return;   // nothing to cut; the counts below divide by the stages
    const int blocks = (P + AT_KEYS - 1) / AT_KEYS;
    const long long HK = (long long)KH * ngc, stages = (long long)B * HK * ((max_len + OWN_KEYS - 1) / OWN_KEYS);
    // The SMs' shares and the prefix's pieces: those whose end is earliest by
    // this count (us, measured at head_dim 128 / 64).  A piece takes 1.9 / 1.1 a
    // block of two tiles and 8 for its start and end; the own keys 8, and an SM
    // 1.1 / 0.9 a stage and 1.7 a sequence and head, no faster than HBM, after
    // which their SMs take pieces too.  The lengths are on the device: caches
    // count as three quarters full, and a window as none, so that windowed
    // calls are cut as if whole.  Batch 256 on 16,384 keys, counted and measured
    // ends: with up to 1,024 own keys 131 and 131 us with 72 SMs and 2 pieces,
    // 181 and 171 with 78 and 3, 233 and 211 with 90 and 2; with up to 256
    // 108 and 105 with 72 and 6, 140 and 149 with 32 and 4.
    own_ctas = max_len > 0 ? (int)std::min((long long)sms, stages) : 0;
    const double tb = HD == 128 ? 1.9 : 1.1, ts = 0.75 * (HD == 128 ? 1.1 : 0.9), th = 0.75 * OWN_KEYS * HD * 4 / 6.0e6;
    const int step = std::max(1, sms / 8), most = max_len > 0 && blocks ? std::max(1, sms - step) : 0;
    double best = 0;
    for (int own = std::min(most, step); blocks && own <= most; own += step) {
      const double free = most ? 8 + std::max((ts * stages + 1.7 * B * HK) / std::min((long long)own, stages), th * stages) : 0;
      for (int n : {1, 2, 3, 4, 5, 6, 8, 12, 16, 32, 64}) {
        if (n > blocks) break;
        const double d = tb * ((blocks + n - 1) / n) + 8;
        const long long m = (long long)units * KH * n;
        const double about = std::max(0.0, (m * d + own * free) / sms);
        double one = std::floor(about / d) * d, two = free + std::max(0.0, std::floor((about - free) / d)) * d;   // both groups' ends
        long long done = (long long)(one / d + 0.5) * (sms - own) + (long long)((two - free) / d + 0.5) * own;
        double end = std::max(one, done > 0 && two > free ? two : 0.0);
        while (done < m) {
          if (!own || one <= two)
            end = std::max(end, one += d), done += sms - own;
          else
            end = std::max(end, two += d), done += own;
        }
        end = std::max(end, free) + 0.5 * n;
        if (!nsp || end < best) {
          best = end, nsp = n;
          if (most) own_ctas = (int)std::min((long long)own, stages);
        }
      }
    }
  }
};

}  // namespace tg
