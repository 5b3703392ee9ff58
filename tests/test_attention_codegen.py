"""The attention kernel with its products in inline asm (attention_tiles.h), checked on the gfx950 code that this build compiles
(CPU only: hipcc -S, no GPU).

The compiler does not see that those instructions are MFMAs, so it puts no wait between one and whatever else uses its
result: the source does. The results' way is followed through every branch of the compiled kernel:
  * no instruction but an MFMA that accumulates in place reads or writes a register within 19 wait states of the MFMA that
    wrote it (the longest that any MFMA needs; an instruction counts one, s_nop its number, an MFMA 7: those of
    32x32x16 follow each other at 8 at the least). That covers copies which the compiler makes;
  * an MFMA's sources are not among the results still on their way, nor written by another vector instruction fewer than two
    wait states before it (values from LDS and memory have their own waits);
  * no scratch is used."""

import re
import subprocess

import pytest

STATES = 19


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    import __graft_entry__

    b = __graft_entry__.load_build_module()
    outs = [tmp_path_factory.mktemp("asm") / f"{n}.s" for n in ("attention_f16", "attention_bf16")]
    procs = [subprocess.Popen([b._hipcc(), *b.HIP_FLAGS, "--cuda-device-only", "-S", str(b.CSRC / f"{o.stem}.hip"), "-o", str(o)],
                              stderr=subprocess.PIPE, text=True) for o in outs]
    found = {}
    for proc, out in zip(procs, outs):
        err = proc.communicate(timeout=900)[1]
        assert proc.returncode == 0, err[-2000:]
        text = out.read_text()
        for m in re.finditer(r"^(_Z\w*attention_tile_kernel\w+):.*?^\.Lfunc_end\d+:", text, re.M | re.S):
            found[m.group(1)] = m.group(0), re.search(rf"\.amdhsa_kernel {m.group(1)}\n(.*?)\.end_amdhsa_kernel", text, re.S).group(1)
    return found


def registers(operand):
    """Names of the vector and accumulation registers in an operand."""
    m = re.match(r"([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m.group(1), r) for r in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"([va])(\d+)\b", operand)
    return {(m.group(1), int(m.group(2)))} if m else set()


def blocks(body):
    """label -> (instructions, labels that may follow); instructions are (name, operands)."""
    out, label, seq, ends = {}, "entry", [], []
    for line in body.split(".Lfunc_end")[0].splitlines()[1:]:
        s = line.split(";")[0].strip()
        m = re.match(r"(\.LBB\w+):", s)
        if m:
            out[label] = (seq, ends + [m.group(1)])
            label, seq, ends = m.group(1), [], []
            continue
        if not s or s.startswith(".") or s.endswith(":"):
            continue
        name, _, rest = s.partition(" ") if " " in s else s.partition("\t")
        ops = [o.strip() for o in rest.split(",")] if rest else []
        if name.startswith("s_cbranch"):
            ends = ends + [ops[-1]]
            out[label] = (seq, ends + [f"{label}+"])
            label, seq, ends = f"{label}+", [], []
        elif name == "s_branch":
            out[label] = (seq, ends + [ops[-1]])
            label, seq, ends = f"{label}+", [], []
        elif name == "s_endpgm":
            out[label] = (seq, ends)
            label, seq, ends = f"{label}+", [], []
        else:
            seq.append((name, ops))
    out[label] = (seq, ends)
    return out


def run(seq, state, complain):
    """state: register -> wait states since an MFMA wrote it, below STATES; ("fresh", register): since another vector
    instruction did, below 2."""
    fresh = {r[1]: n for r, n in state.items() if r[0] == "fresh"}
    state = {r: n for r, n in state.items() if r[0] != "fresh"}
    for name, ops in seq:
        mfma = name.startswith("v_mfma")
        if mfma:
            dst = registers(ops[0])
            for o in ops[1:3]:
                if registers(o) & set(state):
                    complain(f"{name} {ops}: a source is not there yet")
            for o in ops[1:]:
                if registers(o) & set(fresh):
                    complain(f"{name} {ops}: a source is {min(fresh[r] for r in registers(o) & set(fresh))} wait states old")
            if registers(ops[3]) and registers(ops[3]) != dst:
                complain(f"{name} {ops}: not in place")
        elif state:
            for o in ops:
                if registers(o) & set(state):
                    complain(f"{name} {ops}: {min(state[r] for r in registers(o) & set(state))} wait states after the product")
        step = int(ops[0], 0) + 1 if name == "s_nop" else 7 if mfma else 1
        state = {r: n + step for r, n in state.items() if n + step < STATES}
        fresh = {r: n + step for r, n in fresh.items() if n + step < 2}
        if mfma:
            for r in dst:
                state[r] = 0
        elif name.startswith("v_") and not name.startswith("v_cmp"):
            for o in ops[:2] if "swap" in name else ops[:1]:
                fresh.update({r: 0 for r in registers(o)})
    return {**state, **{("fresh", r): n for r, n in fresh.items()}}


def test_kernels_are_found(kernels):
    assert len(kernels) >= 20
    for name, (_, resources) in kernels.items():
        assert re.search(r"\.amdhsa_private_segment_fixed_size 0\b", resources), f"{name} uses scratch"


def test_results_are_waited_for(kernels):
    for name, (body, _) in kernels.items():
        graph = blocks(body)
        assert sum(i[0].startswith("v_mfma") for seq, _ in graph.values() for i in seq) > 20
        entry, todo, bad = {label: {} for label in graph}, ["entry"], set()
        seen = set()
        while todo:
            label = todo.pop()
            seen.add(label)
            seq, follow = graph[label]
            out = run(seq, entry[label], lambda m: bad.add(f"{label}: {m}"))
            for f in follow:
                if f not in graph:
                    continue
                merged = dict(entry[f])
                for r, n in out.items():
                    merged[r] = min(n, merged.get(r, n))
                if merged != entry[f] or f not in seen:
                    entry[f] = merged
                    todo.append(f)
        assert not bad, f"{name}: {sorted(bad)[:5]} ({len(bad)})"


RING = 4  # units of 32 keys that have places in LDS, of keys and of values


def wait_of(ops, counter):
    m = re.search(rf"{counter}\((\d+)\)", " ".join(ops))
    return int(m.group(1)) if m else None


def follow_copies(graph, dim, batch, values, turns=10):
    """Every path of a wave that copies keys, or values, through the compiled kernel, for all numbers of units up to `turns` of its own
    and of the workgroup's. A barrier stands before the first turn and then before every `batch` turns, and all waves run the same
    code between two of them: what lies in LDS behind a barrier is what a wave's wait before it has seen land, and what may be
    overwritten behind it is what turns before it read. Turn u reads the keys of unit u + 1 (those of unit 0 come before the first turn) and the
    values of unit u - 1 (of unit -1, zeros in place 3, at first); behind the last turn the last unit's values are read.
    State: barriers passed, copies issued, landed, landed at the last barrier, reads. Returns (complaints, units read at the ends)."""
    copies, reads = dim // 32, dim // 8 if values else dim // 16  # instructions for a unit
    is_read = "ds_read_b64_tr" if values else "ds_read_b128"
    first = (RING - 2 if values else RING) + 1 - batch  # units copied before the first barrier
    lead = 0 if values else 1
    bad, ends, seen, todo = set(), set(), set(), [("entry", (0, 0, 0, 0, 0))]
    while todo:
        label, state = todo.pop()
        if (label, state) in seen:
            continue
        seen.add((label, state))
        seq, follow = graph[label]
        barriers, issued, landed, ready, read = state
        turn = (barriers - 2) * batch  # the one that the last barrier stands before
        lost = False
        for i, (name, ops) in enumerate(seq):
            if name.startswith("buffer_load") and "lds" in ops[-1].split():
                before = issued // copies - RING  # the unit whose place this copy takes
                if barriers == 0:
                    lost = issued // copies >= RING
                elif before > turn - (2 if values else 0):
                    bad.add(f"{label}: unit {before + RING} is copied over unit {before} behind the barrier of turn {turn}")
                issued += 1
            elif name == "s_waitcnt":
                left = wait_of(ops, "vmcnt")
                if left is not None:
                    landed = max(landed, issued - left)
            elif name == "s_barrier":
                if barriers == 0:
                    lost = issued != first * copies
                else:
                    turn = (barriers - 1) * batch
                    if issued != (turn + first) * copies:
                        bad.add(f"{label}: {issued} copies before turn {turn}")
                    if read >= 0 and read // reads < turn + lead:
                        read = -1  # this wave has fewer units: it has read its last one
                if i == 0 or seq[i - 1][0] != "s_waitcnt" or wait_of(seq[i - 1][1], "lgkmcnt") != 0:
                    bad.add(f"{label}: reads may be on their way at a barrier")
                barriers, ready = barriers + 1, landed
                lost = lost or turn > turns
            elif name.startswith(is_read) and barriers:
                unit = read // reads - (1 if values else 0)
                if read < 0:
                    bad.add(f"{label}: a read behind the last turn's barriers")
                elif (unit + 1) * copies > ready:
                    bad.add(f"{label}: unit {unit} is read behind the barrier of turn {turn}, before which {ready // copies} have landed")
                read += 1 if read >= 0 else 0
            if lost:
                break
        if lost:
            continue
        if not follow and barriers:
            if landed != issued:
                bad.add(f"{label}: copies may be on their way at the end")
            ends.add(read // reads if read >= 0 else -1)
        todo += [(f, (barriers, issued, landed, ready, read)) for f in follow if f in graph]
    return bad, ends


@pytest.mark.parametrize("values", [False, True], ids=["keys", "values"])
def test_copies_are_waited_for(kernels, values):
    """Nothing is read from LDS before its copy has landed and a barrier has told so, nor written over before a barrier behind its
    last read."""
    for name, (body, _) in kernels.items():
        dim, mask = map(int, re.search(r"kernelILi(\d+)ELb\dELi(\d)E", name).groups())
        graph = blocks(body)
        bad, ends = follow_copies(graph, dim, 2 if mask else 1, values)
        assert not bad, f"{name}: {sorted(bad)[:5]} ({len(bad)})"
        # paths of 2, 4, ... units, the first one's values of unit -1 to 1, its keys of unit 0 to 2
        assert {3, 5, 7} <= ends, (name, ends)
