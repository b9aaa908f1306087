"""What the compiler made of the 8-bit product's kernels (kandinsky.cpp_amd/
csrc/kd_f8_mm.hip): f8_mm_tile's products are asm, whose wait states it does
not know, and all three kernels count the DMAs that are on their way."""
import re

import pytest

from kernel_asm import kernels, successors

SOURCE = "kd_f8_mm.hip"


def _regs(text):
    out = set()
    for kind, lo, hi in re.findall(r"\b([av])\[(\d+):(\d+)\]", text):
        out |= {kind + str(r) for r in range(int(lo), int(hi) + 1)}
    return out | {k + r for k, r in re.findall(r"\b([av])(\d+)\b", text)}


def _named(part):
    return [n for n in kernels(SOURCE) if part in n]


def test_every_kernel_is_here():
    assert len(_named("f8_mm_tile")) == 1 and len(_named("f8_mm_ring")) == 10 and len(_named("f8_mm_grid")) == 7


@pytest.mark.parametrize("source", [SOURCE, "kd_f8_rows.hip"])
def test_no_spills_and_no_packed_f32(source):
    for name, lines in kernels(source).items():
        bad = [ln for ln in lines if re.match(r"scratch_|v_pk_(add|mul|fma)_f32", ln)]
        assert not bad, (name, bad[:3])


def test_every_dma_has_its_wait_state_behind_m0():
    for name, lines in kernels(SOURCE).items():
        for i, ln in enumerate(lines):
            if ln.startswith("global_load_lds"):
                assert lines[i - 1] == "s_nop 0", (name, i, lines[i - 2:i + 1])


def test_tile_accumulators_wait_for_the_products():
    """On every path nothing but products touches an accumulator between the
    first product and the wait behind the last (each passes that wait by a
    marker of its own, which the compiler cannot read it ahead of)."""
    lines = kernels(SOURCE)[_named("f8_mm_tile")[0]]
    nxt = successors(lines)
    mfma = [i for i, ln in enumerate(lines) if ln.startswith("v_mfma")]
    acc = set().union(*(_regs(lines[i].split(", ")[0]) for i in mfma))
    assert len(acc) == 256 and all(r[0] == "a" for r in acc)
    marks = [i for i, ln in enumerate(lines) if ln == "; accumulator complete"]
    assert len(marks) == 64
    todo, seen, met = [(j, False) for i in mfma for j in nxt[i]], set(), set()
    while todo:
        i, waited = todo.pop()
        if (i, waited) in seen:
            continue
        seen.add((i, waited))
        ln = lines[i]
        if ln == "; accumulator complete":
            assert waited
            met.add(i)
            if i == marks[-1]:
                continue
        elif ln == "s_nop 15":
            waited = True
        elif ln.startswith("v_mfma"):
            waited = False
        else:
            assert waited or ln.startswith(";") or not _regs(ln) & acc, f"line {i}: {ln}"
        todo += [(j, waited) for j in nxt[i]]
    assert met == set(marks)


def test_tile_operands_are_not_written_just_ahead_of_a_product():
    """No vector instruction writes an operand, scales among them, within four
    wait states ahead of the product that reads it."""
    lines = kernels(SOURCE)[_named("f8_mm_tile")[0]]
    before = {}
    for i, js in enumerate(successors(lines)):
        for j in js:
            before.setdefault(j, []).append(i)
    for i, ln in enumerate(lines):
        if not ln.startswith("v_mfma"):
            continue
        operands, todo, seen = _regs(ln), [(p, 0) for p in before[i]], set()
        while todo:
            j, states = todo.pop()
            if (j, states) in seen:
                continue
            seen.add((j, states))
            up = lines[j]
            if up.startswith("v_") and not up.startswith(("v_mfma", "v_cmp")):
                wrote = _regs(up.split(", ")[0]) | (_regs(up) if "swap" in up else set())
                assert not wrote & operands, f"line {j}: {up} ahead of {ln}"
            nop = re.match(r"s_nop (\d+)", up)
            states += 0 if up.startswith((";", ".")) else int(nop.group(1)) + 1 if nop else 1
            if states < 4:
                todo += [(p, states) for p in before.get(j, [])]


def _steady(lines, products):
    """The lines of the kernel's steady loop, the one of `products` products without conditions."""
    at = {ln[:-1]: i for i, ln in enumerate(lines) if ln.startswith(".L") and ln.endswith(":")}
    for i, ln in enumerate(lines):
        m = re.match(r"s_c?branch\w*\s+(\.L\w+)", ln)
        if m and m.group(1) in at and at[m.group(1)] < i:
            body = lines[at[m.group(1)]:i]
            if sum(b.startswith("v_mfma") for b in body) == products and not any(b.startswith("v_cndmask") for b in body):
                return body
    raise AssertionError("no such loop")


def test_tile_steps_count_their_dmas():
    """Four steps: 64 products and 16 DMAs each, and one wait that leaves the 8
    DMAs of X's latest stage."""
    body = _steady(kernels(SOURCE)[_named("f8_mm_tile")[0]], 256)
    assert sum(b.startswith("global_load_lds_dwordx4") for b in body) == 64
    assert sum(b == "s_barrier" for b in body) == 4
    waits = [b for b in body if b.startswith("s_waitcnt vmcnt(8)")]
    assert len(waits) == 4
    # behind a wait come W's 8 DMAs, then X's 8, up to the next
    kinds = [b for b in body if b.startswith(("global_load_lds", "s_waitcnt vmcnt(8)"))]
    first = kinds.index(waits[0])
    assert [len(list(g)) for g in _runs(kinds[first:])][:6] == [1, 16, 1, 16, 1, 16]


def _runs(kinds):
    run = []
    for k in kinds:
        if run and k.split()[0] != run[-1].split()[0]:
            yield run
            run = []
        run.append(k)
    yield run


@pytest.mark.parametrize("nb,mb,stages,lines", [(4, 2, 5, 0), (4, 3, 5, 0), (4, 5, 4, 0), (4, 8, 3, 0), (4, 2, 5, 1), (4, 3, 5, 1), (4, 5, 4, 1)])
def test_grid_steps_count_their_dmas(nb, mb, stages, lines):
    """Four steps: a wait that leaves what was sent behind the next stage (the
    next two, where a block's chunks lie in two lines), the stages' DMAs and,
    once, a word's."""
    name = [n for n in _named("f8_mm_grid") if f"ILi{nb}ELi{mb}ELi{stages}ELb{lines}E" in n]
    assert len(name) == 1
    body = _steady(kernels(SOURCE)[name[0]], 4 * nb * mb)
    per, word = nb + mb, (32 * (nb + mb) + 255) // 256
    assert sum(b.startswith("global_load_lds_dwordx4") for b in body) == 4 * per
    assert sum(b.startswith("global_load_lds_dword ") for b in body) == word
    assert sum(b == "s_barrier" for b in body) == 4
    left = [int(re.match(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)", b).group(1)) for b in body if re.match(r"s_waitcnt vmcnt\(\d+\) lgkmcnt\(0\)", b)]
    want = [sum(per + (word if (q + t) % 4 == 0 else 0) for t in range(2 + lines, stages)) for q in range(4)]
    assert left == want


@pytest.mark.parametrize("nb,mb,stages,lines", [(1, 1, 4, 0), (2, 2, 4, 0), (4, 1, 3, 0), (4, 2, 3, 0), (4, 5, 1, 0), (1, 1, 4, 1), (2, 2, 4, 1),
                                                (4, 1, 3, 1), (4, 2, 3, 1), (4, 5, 2, 1)])
def test_ring_steps_count_their_dmas(nb, mb, stages, lines):
    """A step's wait leaves the later stages' DMAs (but the next one's, where a
    block's chunks lie in two lines); a stage and what stands in for one are as
    many."""
    name = [n for n in _named("f8_mm_ring") if f"ILi{nb}ELi{mb}ELi{stages}ELb{lines}E" in n]
    assert len(name) == 1
    asm = kernels(SOURCE)[name[0]]
    per = 2 * (nb + mb)
    dmas = sum(ln.startswith("global_load_lds_dwordx4") for ln in asm)
    # ahead of a run and in its step, a stage or its stand-in (a run's first stage is always there)
    assert dmas in [2 * per * (stages + 1) - sure * per for sure in range(2 + lines)]
    assert f"s_waitcnt vmcnt({(stages - 1 - lines) * per})" in asm
