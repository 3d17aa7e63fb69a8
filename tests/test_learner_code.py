"""The learner library's device code as it was built (drloco_amd/csrc/libdrloco_learner.so, disassembled): waits that a missing line would leave out
without any test on the device failing for certain."""
import os
import re
import shutil
import subprocess

import pytest

from drloco_amd import learner_lib as ll

OBJDUMP = shutil.which('llvm-objdump') or '/opt/rocm/llvm/bin/llvm-objdump'


@pytest.fixture(scope='module')
def listing(tmp_path_factory):
    if not os.path.exists(OBJDUMP):
        pytest.skip('no llvm-objdump')
    if not os.path.exists(ll.LIB_PATH):
        ll.build()
    at = tmp_path_factory.mktemp('code')
    shutil.copy(ll.LIB_PATH, at / 'l.so')
    subprocess.run([OBJDUMP, '--offloading', 'l.so'], cwd=at, check=True, capture_output=True)
    code, = [f for f in os.listdir(at) if 'gfx950' in f]
    return subprocess.run([OBJDUMP, '-d', code], cwd=at, check=True, capture_output=True, text=True).stdout


def undrained(text):
    """Barriers that are reached in straight line from a store which other dies may read, with no wait for it in between."""
    bad, open_ = [], False
    for n, line in enumerate(text.splitlines()):
        op = line.split('//')[0].strip()
        if re.match(r'(global|flat|buffer)_store\S* .*\bsc1\b', op):
            open_ = True
        elif re.match(r's_waitcnt\b.*vmcnt\(0\)', op):
            open_ = False
        elif op.startswith('s_barrier') and open_:
            bad.append(n)
        elif re.match(r's_(branch|endpgm|setpc)', op):
            open_ = False
    return bad


def function(listing, part):
    return [f for f in re.split(r'\n(?=[0-9a-f]+ <)', listing) if part in f.split('\n', 1)[0] and '.kd' not in f.split('\n', 1)[0]]


def test_the_checker_on_small_listings():
    store, wait, barrier = 'global_store_dwordx2 v[6:7], v[2:3], off sc1 // 0: 1\n', 's_waitcnt vmcnt(0) // 0: 1\n', 's_barrier // 0: 1\n'
    assert undrained(store + barrier) and undrained(wait + store + 's_waitcnt vmcnt(1)\n' + barrier)
    assert not undrained(store + wait + barrier) and not undrained(store.replace(' sc1', '') + barrier) and not undrained(store + 's_endpgm\n' + barrier)


def test_split_sums_have_arrived_before_they_are_counted(listing):
    """k_orth_direct's Gram form: the waves that leave a share of a split sum wait for their own stores in front of the barrier behind which one of them counts the share."""
    gram, = function(listing, 'k_orth_directILi0E')
    assert re.search(r'global_store_dwordx2 .*sc1', gram) and 'global_atomic_add' in gram
    assert undrained(gram) == []
