"""Linear attention: the 64-bit form against the closed sum, and refusals before anything is launched (no GPU)."""
import math
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")
import linear_reference as ref  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20


def test_the_reference_is_the_sum_over_earlier_tokens():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(9, h, d, generator=g) for h, d in ((2, 5), (2, 5), (4, 3)))
    decay = -torch.rand(9, 4, generator=g)
    states = torch.randn(2, 4, 5, 3, generator=g)
    starts, src, dst = torch.tensor([0, 6, 9]), torch.tensor([1, -1]), torch.tensor([0, 7])
    out, tol, new, _ = ref.linear(q, k, v, decay, starts, None, states, src, dst, 0.5)
    for first, end, S in ((0, 6, states[1].double()), (6, 9, torch.zeros(4, 5, 3).double())):
        for t in range(first, end):
            for h in range(4):
                o = q[t, h // 2].double() @ S[h] * math.exp(decay[first:t + 1, h].double().sum())
                for j in range(first, t + 1):
                    w = math.exp(decay[j + 1:t + 1, h].double().sum())
                    o = o + w * (q[t, h // 2].double() @ k[j, h // 2].double()) * v[j, h].double()
                assert torch.allclose(out[t, h], 0.5 * o, rtol=1e-12, atol=1e-12)
    assert torch.equal(new[1], states[1].double()) and not torch.equal(new[0], states[0].double())
    assert bool((tol > 0).all()) and tol.max() < 1e-3
    cut = ref.linear(q, k, v, decay, starts, 2, states, src, dst, 0.5)[0]
    assert torch.equal(cut[:2], out[:2]) and bool((cut[2:6] == 0).all())


def args(pkg, **over):
    f = dict(q=FAKE, k=FAKE, v=FAKE, decay=FAKE, starts=FAKE, states=FAKE, src=FAKE, dst=FAKE, out=FAKE, qs=256, ks=256,
             vs=512, ds=0, slots=2, seqs=2, total=9, most_q=5, heads=4, hk=2, dk=128, dv=128, it=1, ot=1, scale=1.0)
    f.update(over)
    return pkg._LINEAR.pack(*f.values()) + bytes(4)


BAD = [dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(decay=0), dict(starts=0), dict(q=FAKE + 8), dict(v=FAKE + 2),
       dict(states=0), dict(states=FAKE + 4), dict(slots=-1), dict(slots=1 << 31), dict(qs=248), dict(qs=260), dict(ks=128),
       dict(vs=256), dict(vs=516), dict(ds=3), dict(ds=-1), dict(seqs=-1), dict(total=-1), dict(total=1 << 31),
       dict(most_q=0), dict(most_q=1 << 31), dict(heads=0), dict(heads=5), dict(hk=0), dict(hk=3), dict(dk=0), dict(dv=-64),
       dict(it=3), dict(it=-1), dict(ot=3), dict(scale=math.nan)]


def test_refusals_before_launch(pkg):
    L, E = pkg.lib(), pkg.ERROR_INVALID_VALUE
    for over in BAD:
        a = args(pkg, **over)
        assert L.iq4xs_linear_attention_workspace_bytes(a) == 0, over
        assert L.iq4xs_linear_attention(a, FAKE, 1 << 40, None) == E, over
    assert L.iq4xs_linear_attention(None, FAKE, 1 << 40, None) == E
    for over in (dict(dk=96), dict(dv=32), dict(dk=512), dict(dv=192)):
        assert L.iq4xs_linear_attention(args(pkg, **over), FAKE, 1 << 40, None) == pkg.ERROR_NOT_SUPPORTED, over
    many = args(pkg, heads=1 << 14, hk=1 << 14, qs=1 << 21, ks=1 << 21, vs=1 << 21, seqs=1 << 17, total=1 << 17)
    assert L.iq4xs_linear_attention_workspace_bytes(many) == 0
    assert L.iq4xs_linear_attention(many, FAKE, 1 << 40, None) == pkg.ERROR_INVALID_CONFIG


def test_nothing_to_do_launches_nothing(pkg):
    L = pkg.lib()
    for over in (dict(total=0, q=0), dict(seqs=0)):
        assert L.iq4xs_linear_attention_workspace_bytes(args(pkg, **over)) == 0
        assert L.iq4xs_linear_attention(args(pkg, **over), None, 0, None) == 0


def test_workspaces_too_small_are_refused(pkg):
    """One long sequence of few heads is cut into segments: their states, and what each keeps of the state before it."""
    L, E = pkg.lib(), pkg.ERROR_INVALID_VALUE
    a = args(pkg, seqs=1, total=4096, most_q=4096)
    need = L.iq4xs_linear_attention_workspace_bytes(a)
    assert need >= 2 * 4 * 128 * 128 * 4
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 16, need)):
        assert L.iq4xs_linear_attention(a, ws, size, None) == E, (ws, size)


def test_the_struct_matches_the_header(pkg, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs a host C++ compiler")
    src = tmp_path / "s.cpp"
    src.write_text('#include "iq4xs_mi355x.h"\n#include <cstdio>\nint main() { std::printf("%zu %zu", '
                   'sizeof(iq4xs_linear_attention_args), offsetof(iq4xs_linear_attention_args, scale)); }')
    subprocess.run(["g++", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    size, scale = map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split())
    assert scale + 4 == pkg._LINEAR.size and size >= pkg._LINEAR.size


PLAN = """
#include "linear_plan.h"
#include <initializer_list>
#include <cstdio>
int main() {
    const long long most = 0x7FFFFFFF, lengths[] = {5, 9, 17, 300, 4096, 1 << 30, most - 64, most - 63, most - 1, most};
    for (long long heads : {1LL, 64LL, 1LL << 15}) for (long long seqs : {1LL, 5LL, 1000LL}) for (long long total : lengths)
        for (long long most_q : lengths) for (int type = 0; type < 3; ++type) {
            iq4xs_linear_attention_args g = {};
            g.seqs = seqs, g.total = total, g.most_q = most_q, g.heads = heads, g.dk = g.dv = 128, g.in_type = type;
            iq4xs::LinearPlan p;
            if (!iq4xs::linear_plan(g, 256, p) || p.steps) continue;
            const long long longest = most_q < total ? most_q : total;
            if (p.length < 1 || p.segments < 1 || p.segments > 514 || (long long)p.length * p.segments < longest ||
                (long long)p.length * (p.segments - 1) >= longest || (p.segments > 1 && p.length % 64 != 0))
                std::printf("%lld %lld %lld %lld %d\\n", heads, seqs, total, most_q, type);
        }
}
"""


def test_segments_hold_the_longest_sequence(pkg, tmp_path):
    """Up to the longest that a call may name: none empty, no more than the chip holds at once and what they round up to."""
    if shutil.which("g++") is None:
        pytest.skip("needs a host C++ compiler")
    src = tmp_path / "s.cpp"
    src.write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "qwen_3.8_27b_optimizations_amd", "csrc"), str(src), "-o", str(tmp_path / "s")],
                   check=True)
    r = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True)
    assert r.stdout == ""
