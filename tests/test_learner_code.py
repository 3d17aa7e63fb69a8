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


EMIT = r"""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cmath>
#include <vector>
#define __device__
#define __forceinline__ inline
using std::min;
static struct { int x; } threadIdx;
namespace dlo {
%s
}
// n values of a turned matrix of one column (rows x 1 as the caller sees it): the weight's rows are `apart`, nothing behind its last element may be read
int main(int, char** argv) {
    using namespace dlo;
    const int n = atoi(argv[1]), apart = atoi(argv[2]);
    std::vector<float> out(n, -1.0f), tile(32 * 33);
    std::vector<float> w((size_t)(n - 1) * apart + 1);
    for (size_t i = 0; i < w.size(); ++i) w[i] = i %% std::max(apart, 1) ? 1e6f : 3.0f + (apart ? i / apart : 0);
    product p{};
    p.out = out.data(); p.w = w.data(); p.out_type = p.w_type = 0;
    p.out_at = {n, 1, 1}; p.w_at = {n, 1, apart};
    p.keep = 2.0f; p.gain = SCALE * SCALE; p.m = 1; p.n = n;
    for (int j0 = 0; j0 < n; j0 += 32) {
        for (int i = 0; i < 32; ++i) for (int j = 0; j < 32; ++j) tile[i * 33 + j] = j0 + j;
        for (threadIdx.x = 0; threadIdx.x < 512; ++threadIdx.x) emit<32, 32, 512>(p, 0, tile.data(), 33, 0, j0);
    }
    for (int j = 0; j < n; ++j)
        if (out[j] != 2.0f * w[(size_t)j * apart] + j) { printf("row %%d: %%g\n", j, out[j]); return 1; }
    return 0;
}
"""


@pytest.mark.parametrize('n,apart', [(300, 1), (301, 3), (64, 5), (97, 0)])
def test_the_epilogue_reads_a_weight_where_it_lies(tmp_path, n, apart):
    """A weight of one column whose rows are apart, next to a contiguous result: the epilogue of dl_orth.hpp, compiled for the host with bounds checks."""
    clang = shutil.which('clang++') or '/opt/rocm/llvm/bin/clang++'
    if not os.path.exists(clang):
        pytest.skip('no clang++')
    text = open(os.path.join(ll.CSRC, 'dl_orth.hpp')).read()
    parts = [re.search(pattern, text, re.S).group(0) for pattern in (
        r'typedef _Float16 half8.*?constexpr int FRAG[^\n]*\n', r'struct matrix \{.*?\n\};\n', r'template <typename E> __device__ __forceinline__ float load_as.*?(?=\n// ---- the sum of squares)',
        r'struct product \{.*?\n\};\n', r'template <int I, int J, int THREADS>\n__device__ __forceinline__ void emit.*?\n\}\n')]
    source, program = tmp_path / 'emit.cpp', tmp_path / 'emit'
    source.write_text(EMIT.replace('#include <vector>', '#include <cstdlib>\n#include <vector>') % '\n'.join(parts))
    subprocess.run([clang, '-std=c++17', '-O1', '-g', '-fsanitize=address', '-w', str(source), '-o', str(program)], check=True)
    done = subprocess.run([str(program), str(n), str(apart)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr[-1500:]
