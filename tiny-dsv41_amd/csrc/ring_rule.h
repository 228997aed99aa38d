// ring_rule.h — how many of a wave's loads ring_kernel (inthead.hip) may leave in flight, at each stage and before it reads a
// block's scales.  Loads come back in order, so a wait for all but the youngest n is a wait for the others.  Plain C++: the
// host tests compile it.
//
// A wave's loads, `loads` a stage: those of RING - 1 stages; then at every stage a wait and a barrier, at a block's first one the
// load of the block's scales, and those of the stage RING - 1 further on.
#pragma once

namespace dsv41 {

constexpr int RING = 3;  // stages in LDS (32 tokens a stage, and four stages: no faster)

// At a stage: all but the RING - 2 stages behind it.
constexpr int stage_wait(int loads) { return (RING - 2) * loads; }

// Behind a block of `stages`: all but those of its stages, which were issued after the scales.  -1: the block's last stage
// waited for them.
constexpr int scales_wait(int stages, int loads) { return stages < RING - 1 ? stages * loads : -1; }

}  // namespace dsv41
