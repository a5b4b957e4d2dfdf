"""The wide form of paged_attention_kernel in the built library: its ring of direct-to-LDS loads lies where the
rows of O go once the last step is done, and every wavefront loads into all of it. A step's barrier leaves a step's
loads of each wavefront in flight, so that between the last of them and the stores of O every wavefront must wait
for its own loads and then for the others. Read from the kernel's instructions, since loads are hardly ever late
enough for a run's results to show it."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
SYNC = re.compile(r"s_waitcnt .*vmcnt\((\d+)\)|(s_barrier)|(global_load_lds)|(ds_write_b128)|(s_cbranch\w*|s_branch)\s+(L\d+)|(s_endpgm|s_setpc_b64)")


@pytest.fixture(scope="module")
def kernels(hip, tmp_path_factory):
    """{head_dim, q type: basic blocks by label} of paged_attention_kernel: the instructions that matter here, and
    where each block goes on."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    at = tmp_path_factory.mktemp("ring")
    lib = shutil.copy(hip.LIB._name, at / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=at, check=True, capture_output=True)
    found = {}
    for f in sorted(at.glob("lib.so.*gfx950")):
        if b"paged_attention_kernel" not in f.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--symbolize-operands", str(f)], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <(?=_Z)", text, flags=re.M)[1:]:
            m = re.search(r"paged_attention_kernelILi(\d+)ELb(\d)E", part.split("\n", 1)[0])
            if m:
                found[int(m[1]), int(m[2])] = blocks_of(part)
    return found


def blocks_of(text):
    label, blocks, order = "", {"": ([], [])}, [""]
    for line in text.split("\n")[1:]:
        m = re.match(r"(?:[0-9a-f]+ )?<(L\d+)>:", line)
        if m:
            label = m[1]
            order.append(label)
            blocks[label] = ([], [])
            continue
        m = SYNC.search(line.split("//")[0])
        if not m:
            continue
        ops = blocks[label][0]
        if m[1] is not None:
            ops.append(f"wait {m[1]}")
        elif m[5]:
            # a branch in a block's middle: the rest of it is a block of its own
            blocks[label][1].append(m[6])
            if m[5] != "s_branch":
                label = f"{label}+"
                blocks[order[-1]][1].append(label)
                order.append(label)
                blocks[label] = ([], [])
        else:
            ops.append(next(x for x in (m[2], m[3], m[4], m[7]) if x))
            if m[7]:
                label = f"{label}!"  # nothing follows
                blocks[label] = ([], [])
                order.append(label)
    ended = lambda n: blocks[n][1] or (blocks[n][0] and blocks[n][0][-1] in ("s_endpgm", "s_setpc_b64"))  # noqa: E731
    for a, b in zip(order, order[1:]):
        if not ended(a):
            blocks[a][1].append(b)
    return blocks


@pytest.mark.parametrize("d,q_f16", [(128, 0), (128, 1), (64, 0), (64, 1)])
def test_ring_is_at_rest_before_o_is_stored(kernels, d, q_f16):
    blocks = kernels[d, q_f16]
    loads, stores = 2 * 8 * 2 * d // 1024, d // 8  # a wavefront's loads of a step, and its stores of O
    runs = [n for n, (ops, _) in blocks.items() if ops.count("ds_write_b128") >= stores]
    assert len(runs) >= 2  # both forms store O
    steps = [(n, i) for n, (ops, _) in blocks.items() for i in range(1, len(ops))
             if ops[i] == "s_barrier" and ops[i - 1] == f"wait {loads}"]
    assert len(steps) >= 3  # the first one, and those of two steps a turn
    rings = 0
    for n, i in steps:
        todo, seen = [(n, i + 1)], set()
        while todo:
            n, i = todo.pop()
            ops, to = blocks[n]
            assert ops[i:].count("ds_write_b128") < stores or "s_barrier" in ops[i:ops.index("ds_write_b128", i)], n
            stop = [x for x in ops[i:] if x in ("s_barrier", "global_load_lds")]
            rings += stop[:1] == ["global_load_lds"]
            if not stop:
                todo += [(t, 0) for t in to if t not in seen]
                seen.update(to)
    assert rings  # the walk came through the ring's own loads
