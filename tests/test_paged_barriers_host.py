"""The barriers between the roles of the paged attention's chunk kernel, as a model on the CPU.

A wait on an mbarrier names a phase by its parity: it passes while the phase in progress has the other parity.  It therefore means
what it says only if the barrier can be neither one phase behind nor one phase ahead of what the waiting role expects.  Every role is a
sequence of waits and arrivals, so how far the others can come while one stands still does not depend on the order of steps: for each
wait the model lets all others run as far as they can, and in every order of priorities lets the role come there as early as it can."""
import itertools
import os
import re

import pytest

from conftest import CSRC


def stages(nh, e4m3):
    with open(os.path.join(CSRC, "attention_paged.cu")) as f:
        text = f.read()
    kst, vst = re.search(r"static constexpr int KST = (.+?), VST = (.+?);", text).groups()
    names = {"NH": nh, "E4M3": e4m3}

    def value(c):
        if "?" in c:
            condition, rest = c.split("?", 1)
            yes, no = rest.split(":", 1)
            return value(yes) if eval(condition.replace("||", " or "), dict(names)) else value(no)
        return eval(c, dict(names))

    names["KST"] = value(kst)
    return names["KST"], value(vst), int(re.search(r"static constexpr int RST = (\d+);", text).group(1))


RING = 8                                                    # blocks whose scales the softmax warps may still read


def programs(n, kst, vst, rst, e4m3):
    """("wait", barrier, phase), ("arrive", barrier), ("tensor", barrier): an arrival when the products issued so far are done,
    ("write", block): the block's scales take the place of those of RING blocks before."""
    producer, issuer, converter, groups = [], [], [], [[], []]
    for j in range(n):
        producer += [("wait", "k_empty%d" % (j % kst), j // kst - 1), ("arrive", "k_full%d" % (j % kst))]
        if e4m3:
            producer += [("wait", "raw_empty%d" % (j % rst), j // rst - 1), ("arrive", "raw_full%d" % (j % rst))]
        else:
            producer += [("wait", "v_empty%d" % (j % vst), j // vst - 1), ("arrive", "v_full%d" % (j % vst))]

    def scores(i):
        j, b = i // 2, i % 2
        out = [("wait", "k_full%d" % (j % kst), j // kst)] if b == 0 else []
        out += [("wait", "s_free%d" % b, j - 1), ("tensor", "s_full%d" % b)]
        return out + ([("tensor", "k_empty%d" % (j % kst))] if b == 1 else [])

    issuer += scores(0) + scores(1)
    for i in range(2 * n):
        j, b = i // 2, i % 2
        if i + 2 < 2 * n:
            issuer += scores(i + 2)
        issuer.append(("wait", "p_full%d" % b, j))
        if b == 0:
            issuer.append(("wait", "v_full%d" % (j % vst), j // vst))
        issuer.append(("tensor", "o_full%d" % b))
        if b == 1:
            issuer.append(("tensor", "v_empty%d" % (j % vst)))
    for b in range(2):
        for j in range(n):
            if e4m3:
                groups[b].append(("wait", "ks_full%d" % (j % RING), j // RING))
            groups[b] += [("wait", "s_full%d" % b, j), ("read", j), ("arrive", "s_free%d" % b)]
            if j > 0:
                groups[b].append(("wait", "o_full%d" % b, j - 1))
            groups[b].append(("arrive", "p_full%d" % b))
        groups[b] += [("wait", "o_full0", n - 1), ("wait", "o_full1", n - 1), ("wait", "v_full%d" % ((n - 1) % vst), (n - 1) // vst)]
    if e4m3:
        converter += [("write", 0), ("arrive", "ks_full0")]
        for j in range(n):
            if j + 1 < n:
                converter += [("write", j + 1), ("arrive", "ks_full%d" % ((j + 1) % RING))]
            converter += [("wait", "raw_full%d" % (j % rst), j // rst), ("wait", "v_empty%d" % (j % vst), j // vst - 1),
                          ("arrive", "v_full%d" % (j % vst)), ("arrive", "raw_empty%d" % (j % rst))]
    return [producer, issuer] + groups + ([converter] if e4m3 else [])


class Run:
    def __init__(self, prog):
        self.prog, self.at, self.done = prog, [0] * len(prog), {}
        self.queue, self.read = [], [0, 0]                  # arrivals that wait for the tensor cores; blocks read by each group

    def stands(self, r):
        """The wait that role r stands at: (barrier, phase), or None."""
        op = self.prog[r][self.at[r]] if self.at[r] < len(self.prog[r]) else ("end",)
        return op[1:] if op[0] == "wait" else None

    def check(self):
        for r in range(len(self.prog)):
            w = self.stands(r)
            if w is not None:
                assert self.done.get(w[0], 0) - 1 in (w[1] - 1, w[1]), ("phase", r, w, self.done.get(w[0], 0))

    def step(self, r):
        if self.at[r] == len(self.prog[r]):
            return False
        op = self.prog[r][self.at[r]]
        if op[0] == "wait" and self.done.get(op[1], 0) <= op[2]:
            return False
        if op[0] == "arrive":
            self.done[op[1]] = self.done.get(op[1], 0) + 1
        elif op[0] == "tensor":
            self.queue.append(op[1])
        elif op[0] == "read":
            self.read[r - 2] = op[1] + 1
        elif op[0] == "write":
            assert min(self.read) >= op[1] - RING + 1, ("scales of block %d are still read" % (op[1] - RING),)
        self.at[r] += 1
        self.check()
        return True

    def tensor(self):
        if not self.queue:
            return False
        bar = self.queue.pop(0)
        self.done[bar] = self.done.get(bar, 0) + 1
        self.check()
        return True

    def finish(self, order, frozen=None, until=None):
        """Steps roles (-1: the tensor cores) by priority until nothing moves; `until`: (role, place) to stop at."""
        while True:
            if until is not None and self.at[until[0]] >= until[1]:
                return
            if not any(self.tensor() if r < 0 else r != frozen and self.step(r) for r in order):
                return


@pytest.mark.parametrize("nh,e4m3", [(1, False), (2, False), (1, True), (2, True)])
def test_every_wait_means_the_phase_it_names(nh, e4m3):
    kst, vst, rst = stages(nh, e4m3)
    for n in (1, 2, 3, 7, 12):
        prog = programs(n, kst, vst, rst, e4m3)
        roles = list(range(-1, len(prog)))
        for order in itertools.permutations(roles) if n == 3 else [roles, roles[::-1]]:
            run = Run(prog)
            run.finish(order)
            assert run.at == [len(p) for p in prog] and not run.queue                          # nobody waits for ever
        for r in range(len(prog)):
            for place in range(len(prog[r])):
                run = Run(prog)
                first = [r] + [x for x in roles if x != r]
                run.finish(first, until=(r, place))
                run.finish([x for x in roles if x != r], frozen=r)                              # all others as far as they come
                run.finish(first)
                assert run.at == [len(p) for p in prog]


def test_the_model_finds_what_is_wrong():
    prog = programs(19, 3, 2, 2, True)
    prog[4] = [("arrive", "ks_full0")] * 12 + prog[4]       # a converter that runs ahead
    with pytest.raises(AssertionError):
        Run(prog).finish(range(-1, 5))
    # the halves' products issued independently of one another: a group may be done two blocks before the other
    prog = programs(7, 3, 3, 2, False)
    halves = [[op for op in prog[1] if op[1][-1] == str(b) and op[1][:2] in ("s_", "p_", "o_")] for b in range(2)]
    for j in range(7):
        halves[1].insert(halves[1].index(("wait", "p_full1", j)) + 2, ("tensor", "v_empty%d" % (j % 3)))
        halves[1].insert(halves[1].index(("wait", "s_free1", j - 1)) + 2, ("tensor", "k_empty%d" % (j % 3)))
        halves[0].insert(halves[0].index(("wait", "p_full0", j)), ("wait", "v_full%d" % (j % 3), j // 3))
        halves[0].insert(halves[0].index(("wait", "s_free0", j - 1)), ("wait", "k_full%d" % (j % 3), j // 3))
    prog[1] = halves[0]
    prog.append(halves[1])
    with pytest.raises(AssertionError, match="o_full"):
        for place in range(len(prog[3])):
            run = Run(prog)
            run.finish([3] + [-1, 0, 1, 2, 4], until=(3, place))
            run.finish([-1, 0, 1, 2, 4], frozen=3)
