// fp4_handoff.h - how the warps that copy scales hand steps to the warp that issues the MMAs (fp4_gemm.cu: k_fp4_gemm_wide). Plain
// C++, so that a check on the host can try every order of events with the rule the kernel has.
//
// Step i belongs to copying warp i % CP. When its operands are there the warp arrives at the named barrier of stage i % STAGES and
// goes on; the issuer meets it there. Such a barrier counts arrivals, not steps, so the arrival for step i must not reach it
// before the issuer has been there for step i - STAGES: else two copying warps complete the barrier between them, and the issuer
// waits at the next one for good. While all is well this follows from the wait for the MMAs of step i - STAGES. A warp
// whose wait gave up does not know that any more.
#pragma once

namespace hn {
namespace fp4g {

struct Handoff {
    static constexpr int STAGES = 5;    // of codes, and named barriers
    static constexpr int CP = 4;        // warps that copy scales
    // how many steps the issuer has to have taken before a warp whose wait gave up may arrive for step i
    static constexpr int taken_before(int i) { return i - STAGES + 1; }
};

} // namespace fp4g
} // namespace hn
