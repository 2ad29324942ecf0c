// A ring of pipeline stages as the role that fills it walks it: which stage
// comes next, and the parity of the phase that its barriers complete with that
// fill (an mbarrier's phases alternate 0, 1, 0, ... with its uses).
// tests/test_fp8_blocks_calls.py checks the walk on the CPU against barriers
// that count their phases.
#pragma once
#include <stdint.h>

#ifndef RENG_HD
#ifdef __CUDACC__
#define RENG_HD __host__ __device__ __forceinline__
#else
#define RENG_HD inline
#endif
#endif

namespace reng {

struct Ring {
    int stages, stage, filled;  // filled: stages in use, at most all of them
    uint32_t phase;
    RENG_HD explicit Ring(int n) : stages(n), stage(0), filled(0), phase(0) {}
    // Every stage is in use: the next one's last fill (parity phase ^ 1) has
    // to be consumed first.
    RENG_HD bool full() const { return filled == stages; }
    RENG_HD void fill() {
        if (filled < stages) filled++;
        if (++stage == stages) stage = 0, phase ^= 1u;
    }
    // One step back, to the newest fill that has not been stepped over: its
    // stage and parity.  False when none is left (each stage's last fill has
    // been named once).
    RENG_HD bool back() {
        if (filled == 0) return false;
        filled--;
        if (stage == 0) stage = stages, phase ^= 1u;
        stage--;
        return true;
    }
};

}  // namespace reng
