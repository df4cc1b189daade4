"""The hand-overs between the roles of a gemm_f8_kernel CTA when a bounded wait gives up, on the CPU.

The kernel's warps meet in mbarriers, whose waits have a limit, and in one named barrier (gate and epilogue warps). A
wait that runs out must end the kernel with its status, whichever wait it is and however far the other roles are: no
role may be left behind in a barrier, and no copy may still be on its way into the shared memory of a CTA that has
ended. `explore` walks every order of the roles' steps of a small CTA (few blocks, two epilogue warps); every bounded
wait may give up at any step. The source check at the end ties the model to the kernel."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCKS, STAGES, BUFFERS, EPI = 4, 2, 2, 2


def explore(release, land, blocks=BLOCKS):
    """Every reachable end of a CTA -> set of faults among {"hang", "copy in flight", "bad block stored"}.

    release: how a TMEM buffer goes back to the MMA warp, "named" (bar.arrive of the epilogue warps, bar.sync of the
    MMA warp, which nothing bounds) or "mbarrier" (a wait that can give up). land: when the producer waits for its
    copies, "own" (where it saw the abort itself) or "all" (behind the CTA's last barrier, whoever aborted).

    State: producer, MMA, gate: block and step; epilogue warps: block; copies landed; MMAs done; TMEM arrivals; abort.
    Completed phases of `empty` and `t_full` follow from the MMAs done (in order)."""
    faults, seen = set(), set()
    # (p, p_done, p_saw, landed, m, m_ok, m_step, done, issued, g, g_ok, waiting, e, released, phase, arrived, bad, abort)
    start = (0, False, False, 0, 0, True, 0, 0, 0, 0, True, 0, (0,) * EPI, 0, (0,) * BUFFERS, (0,) * BUFFERS, False, False)
    stack = [start]
    while stack:
        s = stack.pop()
        if s in seen:
            continue
        seen.add(s)
        (p, p_done, p_saw, landed, m, m_ok, m_step, done, issued, g, g_ok, waiting, e, released, phase, arrived, bad, abort) = s

        def go(**kw):
            d = dict(p=p, p_done=p_done, p_saw=p_saw, landed=landed, m=m, m_ok=m_ok, m_step=m_step, done=done, issued=issued,
                     g=g, g_ok=g_ok, waiting=waiting, e=e, released=released, phase=phase, arrived=arrived, bad=bad, abort=abort)
            d.update(kw)
            stack.append(tuple(d.values()))

        before = len(stack)
        # hardware: a copy lands, an MMA ends
        if landed < p:
            go(landed=landed + 1)
        if done < issued:
            go(done=done + 1)
        # producer: waits for the stage (its MMA, STAGES blocks earlier, is done), then copies
        if not p_done:
            if p == blocks:
                go(p_done=True, p_saw=abort)
            else:
                if p < STAGES or done > p - STAGES:
                    go(p=p + 1)
                go(p_done=True, p_saw=True, abort=True)  # its wait gives up
        # MMA: 0 the stage's copy, 1 the buffer, then issue
        if m < blocks:
            if m_step == 0:
                if not m_ok:
                    go(m_step=1)
                else:
                    if landed > m:
                        go(m_step=1)
                    go(m_step=1, m_ok=False, abort=True)
            else:
                u = m % BUFFERS
                nxt = dict(m=m + 1, m_step=0)
                if release == "named":
                    # bar.sync of EPI + 1 warps: passes in the phase that its own arrival completes
                    if m < BUFFERS:
                        go(**nxt, issued=issued + m_ok)
                    elif arrived[u] >= EPI:
                        a = list(arrived)
                        a[u] -= EPI
                        go(**nxt, issued=issued + m_ok, arrived=tuple(a))
                    # (EPI + 1 arrivals of the epilogue alone complete a phase without it: see below)
                else:
                    if not m_ok:
                        go(**nxt)
                    else:
                        if m < BUFFERS or phase[u] >= m // BUFFERS:
                            if m >= BUFFERS and released < m - BUFFERS + 1 and not abort:
                                faults.add("buffer overwritten")
                            go(**nxt, issued=issued + 1)
                        go(**nxt, m_ok=False, abort=True)
        # gate: a block's sums (block g, in order), then the barrier with the epilogue
        if g < blocks and not waiting:
            if not g_ok:
                go(waiting=1)
            else:
                if done > g:
                    go(waiting=1)
                go(waiting=1, g_ok=False, abort=True)
        if waiting and all(x == g for x in e):  # every epilogue warp is at the barrier: it opens
            go(waiting=0, g=g + 1, bad=bad or not g_ok, released=released)
        # epilogue warps: behind the barrier (gate is past block e[i]) read, release the buffer, next block
        for i in range(EPI):
            if e[i] < g:
                u, x = e[i] % BUFFERS, list(e)
                x[i] += 1
                a, ph = list(arrived), list(phase)
                a[u] += 1
                if release == "named":
                    if a[u] == EPI + 1:  # the barrier's count is full without the MMA warp
                        a[u] = 0
                elif a[u] == EPI:
                    a[u], ph[u] = 0, ph[u] + 1
                go(e=tuple(x), arrived=tuple(a), phase=tuple(ph), released=min(x))
        if len(stack) == before or (p_done and m == blocks and g == blocks and not waiting and min(e) == blocks):
            if not (p_done and m == blocks and g == blocks and not waiting and min(e) == blocks):
                if landed == p and done == issued:
                    faults.add("hang")
                continue
            # all roles are at the CTA's last barrier
            if landed < p and not (p_saw if land == "own" else abort):
                faults.add("copy in flight")
            if bad and not abort:
                faults.add("bad block stored")
    return faults


def test_every_wait_may_give_up():
    assert explore("mbarrier", "all") == set()


@pytest.mark.parametrize("blocks", [1, 2, 3, 5])
def test_other_lengths(blocks):
    assert explore("mbarrier", "all", blocks) == set()


def test_the_model_sees_a_barrier_that_outruns_the_mma_warp():
    """Epilogue warps that do not block arrive twice in one phase: the MMA warp then waits for good."""
    assert "hang" in explore("named", "all")


def test_the_model_sees_copies_that_outlive_the_cta():
    """The MMA warp gives up after the producer has issued its last copy and seen no abort."""
    assert "copy in flight" in explore("mbarrier", "own")


def source():
    with open(os.path.join(ROOT, "feml_b200", "csrc", "kernels", "gemm_f8.cu")) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_the_kernel_has_no_unbounded_hand_over():
    """One named barrier, which the gate and epilogue warps pass in the same number; everything else that waits for
    another role is an mbarrier wait with a limit."""
    text = source()
    assert "bar.arrive" not in text
    assert len(re.findall(r"bar\.sync", text)) == 1 and "bar.red" not in text


def test_the_kernel_lands_its_copies_whoever_aborted():
    """Behind the CTA's last barrier, where the abort flag is final."""
    text = source()
    last = text.index("__syncthreads();", text.index("store_rows<T, C::COLS>("))
    assert "mbar_wait_bounded(&full[" in text[last:]


def test_an_aborted_cta_writes_nan():
    """Output that an aborted CTA could not compute is NaN, never what the buffer held: the stores are not skipped, and
    both the plain and the cluster-split output look at the abort first."""
    text = source()
    assert "!*abort_flag" not in text and "!broken" not in text
    plain = text[:text.index("store_rows<T, C::COLS>(")]
    assert "acc[i] = 0x7fffffff7fffffffull" in plain[plain.rindex("if (*abort_flag)"):]
    split = text[text.index("int broken = 0"):]
    assert "if (broken) f[0] = f[1] = f[2] = f[3] = __int_as_float(0x7fffffff)" in split[:split.index("float4 *>(o)")]
