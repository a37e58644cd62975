// The order of the vector work in a tile of the dK/dV kernels (attn_bwd_mfma.hip, window_attn_bwd.hip).
#ifndef MYFA_ATTN_BWD_PLAN_H_
#define MYFA_ATTN_BWD_PLAN_H_

namespace myfa {
namespace {

// The vector work of one tile of the dK/dV kernel, planned at compile time.
//
// One wave per SIMD means nothing but the wave's own MFMAs can cover its vector instructions, and
// the wave issues ONE instruction at a time: everything that is not an MFMA has to fit, in issue
// slots, between MFMAs that each keep the matrix core busy for 32 cycles.  A tile is 8 KS MFMA
// steps (g = 0 .. 8 KS - 1):
//     A  [0, 2KS)    S0 = Q0 K^T (KS steps), dP0 = dO0 V^T (KS)        block 0 = queries 0..31
//     B  [2KS, 4KS)  S1, dP1                                            block 1 = queries 32..63
//     C  [4KS, 6KS)  dV += dO0^T P0, dK += Q0^T dS0, alternating; its first half takes elements
//                    0..7 of the block's accumulators, its second half elements 8..15
//     D  [6KS, 8KS)  the same for block 1
// and per accumulator element e of a block the vector work is
//     kind 0   t = s * scale*log2e - lse2          (needs S: two steps behind its last MFMA)
//     kind 1   p = exp2(t)
//     kind 2   ds = p * dp                         (needs dP, which started from -delta)
//     kind 3   P pair (2e, 2e+1) -> 16 bit         kind 4   dS pair -> 16 bit
// plan_dkv() deals these 128 operations onto the steps: earliest deadline first, an operation
// never in the same step as the one it depends on, at most `cap` cycles of issue per step.
struct DkvOp { int blk, kind, e; };
template <int KS> struct DkvPlan {
    static constexpr int NSTEP = 8 * KS, NOPS = 128;
    DkvOp op[NOPS] = {};
    int start[NSTEP + 1] = {};
    bool ok = false;
};
template <int KS>
constexpr DkvPlan<KS> plan_dkv(int cap) {
    constexpr int cost[5] = {5, 9, 5, 8, 8};
    DkvPlan<KS> p{};
    int at[2][5][16] = {};
    for (int b = 0; b < 2; ++b)
        for (int k = 0; k < 5; ++k)
            for (int e = 0; e < 16; ++e) at[b][k][e] = -1;
    int n = 0;
    bool late = false;
    for (int g = 0; g < p.NSTEP; ++g) {
        p.start[g] = n;
        int budget = cap;
        while (true) {
            int bb = -1, bk = -1, be = -1, bdl = 1 << 30;
            for (int b = 0; b < 2; ++b) {
                const int s_rdy = (2 * b + 1) * KS + 1, dp_rdy = (2 * b + 2) * KS + 1;
                for (int k = 4; k >= 0; --k)
                    for (int e = 0; e < (k < 3 ? 16 : 8); ++e) {
                        if (at[b][k][e] >= 0) continue;
                        bool rdy = false;
                        if (k == 0) rdy = g >= s_rdy;
                        if (k == 1) rdy = at[b][0][e] >= 0 && at[b][0][e] < g;
                        if (k == 2) rdy = g >= dp_rdy && at[b][1][e] >= 0 && at[b][1][e] < g;
                        if (k == 3) rdy = at[b][1][2 * e] >= 0 && at[b][1][2 * e] < g && at[b][1][2 * e + 1] >= 0 && at[b][1][2 * e + 1] < g;
                        if (k == 4) rdy = at[b][2][2 * e] >= 0 && at[b][2][2 * e] < g && at[b][2][2 * e + 1] >= 0 && at[b][2][2 * e + 1] < g;
                        if (!rdy) continue;
                        const int e0 = k < 3 ? e : 2 * e;
                        const int dl = (4 + 2 * b) * KS + (e0 >= 8 ? KS : 0) - 1;     // last step it may run behind
                        if (dl < bdl) { bdl = dl; bb = b; bk = k; be = e; }           // (ties: later kind, lower element)
                    }
            }
            if (bb < 0 || cost[bk] > budget) break;
            budget -= cost[bk];
            at[bb][bk][be] = g;
            p.op[n++] = DkvOp{bb, bk, be};
            if (g > bdl) late = true;
        }
    }
    p.start[p.NSTEP] = n;
    p.ok = n == p.NOPS && !late;
    return p;
}
// the smallest issue budget per step (in cycles) that meets every deadline
template <int KS, int CAP = 16, bool OK = plan_dkv<KS>(CAP).ok> struct DkvPlanFor;
template <int KS, int CAP> struct DkvPlanFor<KS, CAP, true> {
    static constexpr int cap = CAP;
    static constexpr DkvPlan<KS> plan = plan_dkv<KS>(CAP);
};
template <int KS, int CAP> struct DkvPlanFor<KS, CAP, false> : DkvPlanFor<KS, CAP + 2> {};

}  // namespace
}  // namespace myfa
#endif  // MYFA_ATTN_BWD_PLAN_H_
