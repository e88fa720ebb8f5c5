"""Addresses of the loads in inline asm.  A scalar register that a vector
instruction has written (a readfirstlane, a spilled register's reload) may be
read by a load five wait states later at the earliest; the compiler sees to
that in its own loads, not in inline asm, where an address read too early is
another one's.  The generated code of every source with such loads is searched
for one, straight line by straight line (no GPU)."""
import os
import re
import subprocess

import pytest

from streaming_sparse_amd import build

WAIT = 5
SOURCES = [s for s in build.SOURCES if s == "attention.hip" or s.startswith("paged")]


def early_reads(text):
    """(function, instruction) of each load or store that reads a scalar register
    less than five wait states after a vector instruction wrote it."""
    function, now, written, found = None, 0, {}, []
    for line in text.splitlines():
        label = re.match(r'(_Z\w+):', line)
        if label:
            function, now, written = label.group(1), 0, {}
        code = line.split(';')[0].strip()
        if not code or code.startswith('.') or code.endswith(':'):
            continue
        op, _, rest = code.partition(' ')
        if op == 's_nop':
            now += int(rest, 0) + 1
            continue
        now += 1

        def registers(operand):
            m = re.fullmatch(r's(\d+)|s\[(\d+):(\d+)\]', operand.strip())
            return [] if not m else [int(m[1])] if m[1] else list(range(int(m[2]), int(m[3]) + 1))

        operands = rest.split(',')
        if op.startswith(('global_', 'buffer_', 'flat_', 'scratch_')):
            used = [r for x in operands for part in x.split() for r in registers(part)]
            if any(now - written.get(r, -WAIT) - 1 < WAIT for r in used):
                found.append((function, code))
        elif op.startswith('v_'):
            for x in operands[:2 if '_co_' in op else 1]:
                written.update(dict.fromkeys(registers(x), now))
        elif op.startswith('s_'):
            for r in registers(operands[0]):
                written.pop(r, None)
    return found


def test_an_early_read_is_found():
    start = "_Zkernel:\n\tv_readfirstlane_b32 s5, v0\n"
    load = "\tglobal_load_lds_dwordx4 v1, s[4:5] offset:1024\n"
    assert early_reads(start + load) and early_reads(start + "\ts_nop 3\n" + load)
    assert not early_reads(start + "\ts_nop 4\n" + load)
    assert not early_reads(start + "\ts_add_u32 s5, s6, s7\n" + load)
    assert not early_reads(start.replace('s5', 's6') + load)


def test_no_load_reads_its_address_early(tmp_path):
    try:
        cc = build.hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    runs = []
    for source in SOURCES:
        out = str(tmp_path / source.replace('.hip', '.s'))
        cmd = [cc, *build.FLAGS, *build.EXTRA.get(source, []), '-S', '--offload-device-only', os.path.join(build.CSRC, source),
               '-o', out]
        runs.append((source, out, subprocess.Popen(cmd, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE)))
    for source, out, run in runs:
        err = run.communicate()[1]
        assert run.returncode == 0, err.decode()[-2000:]
        text = open(out).read()
        assert 'global_load_lds' in text, source
        assert not early_reads(text), (source, early_reads(text)[:5])
