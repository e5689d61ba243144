"""Waits behind matrix products, on every way through the compiled kernels.

The hardware does not hold back a vector or memory instruction that uses a
matrix product's result too early: the compiler puts enough instructions or
s_nop between them. It counts them along one way to a place that two lead to
(a product, a short `if`, the use), which may be the longer one. So the
assembly of the linear attention kernels is walked here on all ways: the
shortest one from a product to the first use of its result has to have the
wait states that the compiler itself keeps in straight code, 8 for 16x16x32.
"""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkfft-rs_amd", "csrc")
WAIT = 8


def _registers(text):
    out = set()
    for kind, one, first, last in re.findall(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        out.update((kind, i) for i in (range(int(one), int(one) + 1) if one else range(int(first), int(last) + 1)))
    return out


def _parse(text):
    code, labels = [], {}
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        label = re.match(r"(\S+):$", line)
        if label:
            labels[label[1]] = len(code)
        elif line and not line.startswith("."):
            name, *rest = line.split(None, 1)
            code.append((name, rest[0] if rest else ""))
    return code, labels


def early_uses(text):
    """(product, use, wait states) of each result that is used too early."""
    code, labels = _parse(text)

    def following(i):
        name, rest = code[i]
        if name in ("s_endpgm", "s_setpc_b64"):
            return []
        if name == "s_branch":
            return [labels[rest.strip()]]
        if name.startswith("s_cbranch"):
            return [i + 1, labels[rest.strip()]]
        return [i + 1]

    found = []
    for i, (name, rest) in enumerate(code):
        if not name.startswith("v_mfma"):
            continue
        assert "16x16x32" in name, f"no wait known for {name}"
        result = _registers(rest.split(",")[0])
        least, ways = {}, [(j, 0) for j in following(i)]
        while ways:
            j, passed = ways.pop()
            if j >= len(code) or passed >= WAIT or least.get(j, WAIT) <= passed:
                continue
            least[j] = passed
            use, operands = code[j]
            if use.startswith("v_mfma"):
                to, a, b, c = (_registers(x) for x in operands.split(",")[:4])
                if (a | b) & result or (c & result and c != result):
                    found.append((f"{name} {rest}", f"{use} {operands}", passed))
                if c == result or to & result:
                    continue  # products wait for the ones that they add to
            elif use.startswith(("v_", "ds_", "global_", "flat_", "buffer_", "scratch_")) and _registers(operands) & result:
                found.append((f"{name} {rest}", f"{use} {operands}", passed))
                continue
            states = int(operands, 0) + 1 if use == "s_nop" else 1
            ways += [(k, passed + states) for k in following(j)]
    return found


PRODUCT = "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]\n"
LONG = "".join(f"\tv_mul_f32_e32 v{i}, v40, v{i}\n" for i in range(20, 30))


def test_the_walk_takes_the_shorter_way():
    use = "\tv_mul_f32_e32 v3, v3, v40\n\ts_endpgm\n"
    assert len(early_uses(PRODUCT + "\ts_cbranch_vccnz .L\n" + LONG + ".L:\n" + use)) == 1
    assert not early_uses(PRODUCT + "\ts_cbranch_vccnz .L\n" + LONG + ".L:\n\ts_nop 6\n" + use)
    assert not early_uses(PRODUCT + LONG + use)
    assert len(early_uses(PRODUCT + "\ts_nop 5\n\tv_mov_b32_e32 v41, 0\n" + use)) == 1
    # a product that adds to the result waits for it; one that takes it for a factor does not
    assert not early_uses(PRODUCT + PRODUCT.replace("v[0:3],", "v[4:7],", 1) + "\ts_endpgm\n")
    assert len(early_uses(PRODUCT + PRODUCT.replace("v[8:11]", "v[0:3]").replace("v[0:3],", "v[4:7],", 1) + "\ts_endpgm\n")) == 1


@pytest.mark.skipif(not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="no hipcc")
def test_no_product_is_used_early(tmp_path):
    files = [f"{tmp_path}/linear_{e}.s" for e in ("f32", "f16", "bf16")]
    subprocess.run(["make", "-s", "-j3", "-C", CSRC, f"OBJDIR={tmp_path}"] + files, check=True, capture_output=True, timeout=900)
    kernels = 0
    for f in files:
        text = open(f).read()
        for m in re.finditer(r"^(_Z\S+):\s*; @", text, re.M):
            body = text[m.end():text.index(".Lfunc_end", m.end())]
            if "v_mfma" in body:
                kernels += 1
                assert not early_uses(body), m[1]
    assert kernels >= 60
