"""A randomised CPU model of how the 8-bit products' CTAs come to their end.

``tcgen05.commit`` arrives on an mbarrier some time after it was issued, in shared memory of the CTA and, for a pair of
CTAs, of both. The issuing warp commits an accumulator first and the stage that it was multiplied from second.
Whoever waits for the accumulator has not waited for the stage: the CTA can be gone, and its shared memory
another's, when the release of a stage arrives that no producer waits for. So the issuers of ``fp8_gemm.cuh`` and
``fp8_pair_gemm.cuh`` do not hand the last stages back: those that no later block fills again.

The model runs the producers, the issuer and the summing warps of one or two CTAs with the kernels' index arithmetic
under a random scheduler, lets every commit arrive late by a random time in each CTA, and reports an
arrival in a CTA that has left, a parity test that passes for another phase than the one meant, and deadlock."""
import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tilelang_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


PAIR, TILE = source("fp8_pair_gemm.cuh"), source("fp8_gemm.cuh")
#: whether the issuers keep the last stages, as the sources have it
PAIR_KEEPS = "if (i + kPairStages < blocks) tc_commit_pair(&ctl->empty[s]);" in PAIR
TILE_KEEPS = "if (kb + C::kStages < kb1) tc_commit(&ctl->empty[s]);" in TILE
PAIR_STAGES = int(re.search(r"constexpr int kPairStages = (\d+);", PAIR).group(1))
TILE_STAGES = [int(n) for n in re.search(r"kStages = TN == 32 \? (\d+) : (\d+);", TILE).groups()]
TILE_ACC = int(re.search(r"kAcc = (\d+);", TILE).group(1))


class Violation(Exception):
    pass


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.completed = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.completed, self.pending = self.completed + 1, self.count

    def test(self, parity):
        return (self.completed & 1) != parity


class Model:
    def __init__(self, ctas, stages, accs, blocks, keep, rng):
        self.ctas, self.stages, self.accs, self.blocks, self.keep, self.rng = ctas, stages, accs, blocks, keep, rng
        self.full = [Barrier(ctas) for _ in range(stages)]                       # the first CTA's: both halves have landed
        self.empty = [[Barrier(1) for _ in range(stages)] for _ in range(ctas)]
        self.acc_full = [[Barrier(1) for _ in range(accs)] for _ in range(ctas)]
        self.acc_empty = [Barrier(ctas) for _ in range(accs)]
        self.late = []                                                           # (time, cta, barrier): arrivals on their way
        self.now, self.left = 0, False

    def wait(self, bar, parity, phase):
        while not bar.test(parity):
            yield
        if phase >= 0 and bar.completed != phase + 1:
            raise Violation(f"the test for phase {phase} passed with {bar.completed} phases complete")

    def producer(self, cta):
        s = phase = 0
        for n in range(self.blocks):
            yield from self.wait(self.empty[cta][s], phase ^ 1, n // self.stages - 1)
            self.full[s].arrive()
            s += 1
            if s == self.stages:
                s, phase = 0, phase ^ 1
            yield

    def commit(self, bars):
        for cta, bar in enumerate(bars):
            self.late.append((self.now + self.rng.choice((0, 1, 5, 60)), cta, bar))

    def issuer(self):
        s = phase = 0
        for i in range(self.blocks):
            buf = i % self.accs
            yield from self.wait(self.full[s], phase, i // self.stages)
            yield from self.wait(self.acc_empty[buf], ((i // self.accs) & 1) ^ 1, i // self.accs - 1)
            self.commit([a[buf] for a in self.acc_full])
            if not self.keep or i + self.stages < self.blocks:
                self.commit([e[s] for e in self.empty])
            s += 1
            if s == self.stages:
                s, phase = 0, phase ^ 1
            yield

    def summing(self, cta):
        for i in range(self.blocks):
            buf = i % self.accs
            yield from self.wait(self.acc_full[cta][buf], (i // self.accs) & 1, i // self.accs)
            self.acc_empty[buf].arrive()
            yield

    def run(self):
        roles = [self.issuer()] + [f(c) for c in range(self.ctas) for f in (self.producer, self.summing)]
        speed = [self.rng.choice((1, 1, 6)) for _ in roles]
        while roles or self.late:
            self.now += 1
            for arrival in [a for a in self.late if a[0] <= self.now]:
                self.late.remove(arrival)
                if self.left:
                    raise Violation(f"an arrival in CTA {arrival[1]}, which has left")
                arrival[2].arrive()
            for i in reversed(range(len(roles))):
                if self.rng.randrange(speed[i]) == 0:
                    try:
                        next(roles[i])
                    except StopIteration:
                        del roles[i], speed[i]
            self.left = not roles                                    # the closing barrier: every role of every CTA is done
            if self.now > 200 * (self.blocks + 20):
                raise Violation("deadlock")


KERNELS = [("pair", 2, PAIR_STAGES, 2)] + [("tile", 1, n, TILE_ACC) for n in TILE_STAGES]


def attempts(ctas, stages, accs, keep):
    for seed in range(150):
        rng = random.Random(seed)
        Model(ctas, stages, accs, rng.randrange(3 * stages + 2), keep, rng).run()


@pytest.mark.parametrize("name,ctas,stages,accs", KERNELS)
def test_no_arrival_comes_after_the_end(name, ctas, stages, accs):
    assert PAIR_KEEPS if name == "pair" else TILE_KEEPS
    attempts(ctas, stages, accs, True)


@pytest.mark.parametrize("name,ctas,stages,accs", KERNELS)
def test_with_every_stage_handed_back_one_does(name, ctas, stages, accs):
    with pytest.raises(Violation, match="has left"):
        attempts(ctas, stages, accs, False)
