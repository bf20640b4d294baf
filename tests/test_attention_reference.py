"""The 64-bit reference of the attention tests against closed forms, and the refusals of the attention calls, which touch
no GPU: every call here fails its checks before anything is launched."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import attention_reference as ref  # noqa: E402


def test_reference_of_equal_scores_is_the_mean():
    """Keys of zero: every weight is 1/n, so row i of a causal prompt is the mean of values 0..i."""
    v = torch.arange(5 * 64, dtype=torch.float64).view(5, 64)
    pages = torch.zeros(2, 1, 16, 64)
    pages[1, 0, :5] = v
    o, lse, _, _ = ref.attention(torch.randn(5, 2, 64), torch.zeros(2, 1, 16, 64), pages, None, None,
                           torch.tensor([[1]]), torch.tensor([0, 5]), torch.tensor([5]), True, 0, 0.5)
    for i in range(5):
        assert torch.allclose(o[i], v[:i + 1].mean(0).expand(2, 64))
        assert torch.allclose(lse[i], torch.full((2,), math.log(i + 1), dtype=torch.float64))
    o, lse, _, _ = ref.attention(torch.randn(5, 2, 64), torch.zeros(2, 1, 16, 64), pages, None, None,
                           torch.tensor([[1]]), torch.tensor([0, 5]), torch.tensor([5]), True, 2, 0.5)
    assert torch.allclose(o[4], v[3:5].mean(0).expand(2, 64)) and torch.allclose(o[0], v[0].expand(2, 64))
    # more new tokens than cached ones: the first rows see nothing
    o, lse, _, _ = ref.attention(torch.randn(5, 2, 64), torch.zeros(2, 1, 16, 64), pages, None, None,
                           torch.tensor([[1]]), torch.tensor([0, 5]), torch.tensor([3]), True, 0, 0.5)
    assert (o[:2] == 0).all() and (lse[:2] == -math.inf).all() and torch.allclose(o[4], v[:3].mean(0).expand(2, 64))


def test_reference_rotation_keeps_norms_and_differences():
    """Rotation keeps a pair's length, and the product of two turned rows depends on the difference of positions."""
    g = torch.Generator().manual_seed(3)
    x, f = torch.randn(4, 1, 64, generator=g), ref.frequencies(64)
    for half in (True, False):
        at = lambda p: ref.norm_rope(x, torch.tensor([p] * 4), f, None, 0.0, half)  # noqa: E731
        assert torch.allclose(at(70001).square().sum(-1), torch.full((4, 1), 64.0, dtype=torch.float64))
        a, b = (at(5) * at(2).flip(0)).sum(-1), (at(100005) * at(100002).flip(0)).sum(-1)
        assert torch.allclose(a, b, atol=1e-8)
        assert torch.equal(at(0), ref.norm_rope(x, None, None, None, 0.0, half))


def test_reference_codes_round_trip():
    x = torch.randn(7, 3, 64) * torch.logspace(-6, 6, 7)[:, None, None]
    x[0, 0] = 0
    q, d = ref.codes(x)
    back = ref.stored(q, d)
    lim = x.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).clamp(max=65504)
    err = (back - x.double().clamp(-65504, 65504)).unflatten(-1, (-1, 32)).abs()
    # half a step of the scale, which itself is off by half an fp16 step (or a subnormal's)
    assert (err <= lim * (0.5 / 127 + 2.0 ** -11) + 127 * 2.0 ** -25).all()


FAKE = 0x100000  # never dereferenced


def cache_of(pkg, **over):
    f = dict(k=FAKE, v=FAKE, ks=0, vs=0, pages=4, heads=2, page=16, d=128, type=pkg.TYPE_F16)
    f.update(over)
    return ctypes.create_string_buffer(pkg._CACHE.pack(*f.values()), pkg._CACHE.size)


def test_struct_sizes_match_the_header(pkg, tmp_path):
    import os
    import shutil
    import subprocess

    if shutil.which("g++") is None:
        pytest.skip("needs a host C++ compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.cpp"
    src.write_text('#include "iq4xs_mi355x.h"\n#include <cstdio>\nint main() { std::printf("%zu %zu %zu %zu %zu", '
                   "sizeof(iq4xs_kv_cache), sizeof(iq4xs_qk_norm_rope_args), sizeof(iq4xs_paged_attention_args), "
                   "offsetof(iq4xs_qk_norm_rope_args, eps), offsetof(iq4xs_paged_attention_args, scale)); }")
    subprocess.run(["g++", "-I" + os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    a, b, c, eps, scale = map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split())
    assert (a, b, eps + 4, scale + 4) == (pkg._CACHE.size, pkg._QK.size, pkg._QK.size, pkg._ATTENTION.size)
    assert c >= pkg._ATTENTION.size


BAD_CACHES = [dict(k=0), dict(v=FAKE + 8), dict(pages=0), dict(pages=1 << 28), dict(heads=0), dict(page=24),
              dict(page=8), dict(page=0), dict(type=0), dict(type=9), dict(type=3), dict(type=3, ks=FAKE), dict(d=0)]


def qk_args(pkg, **over):
    f = dict(q=FAKE, k=FAKE, v=FAKE, qs=512, ks=256, vs=256, pos=FAKE, freqs=FAKE, gq=0, gk=0, slots=FAKE, qo=FAKE,
             ko=FAKE, tokens=3, hq=4, hk=2, d=128, rot=128, rope=0, it=0, ot=1, eps=1e-6)
    f.update(over)
    return pkg._QK.pack(*f.values())


BAD_QK = [dict(q=0), dict(k=0), dict(q=FAKE + 4), dict(qs=504), dict(ks=257), dict(pos=0), dict(freqs=0), dict(qo=0),
          dict(tokens=-1), dict(tokens=1 << 31), dict(hq=0), dict(hk=0), dict(rot=144), dict(rot=-16), dict(rope=2),
          dict(it=3), dict(ot=3), dict(it=-1), dict(eps=-1.0), dict(eps=math.nan), dict(gq=FAKE + 2)]


def attention_args(pkg, of, **over):
    f = dict(q=FAKE, out=FAKE, lse=0, cache=ctypes.addressof(of), table=FAKE, starts=FAKE, kv=FAKE, qs=512, width=2,
             seqs=1, total=3, most_q=3, most_kv=20, window=0, hq=4, type=1, ot=1, causal=1, scale=0.1)
    f.update(over)
    return pkg._ATTENTION.pack(*f.values()) + bytes(4)


BAD_ATTENTION = [dict(q=0), dict(out=0), dict(cache=0), dict(table=0), dict(starts=0), dict(kv=0), dict(qs=256),
                 dict(qs=516), dict(width=0), dict(total=-1), dict(seqs=-1), dict(total=1 << 31), dict(most_q=0),
                 dict(most_kv=0), dict(window=-1), dict(hq=5), dict(hq=0), dict(type=0), dict(type=2), dict(type=3),
                 dict(ot=3), dict(scale=math.nan), dict(q=FAKE + 2)]


def test_refusals_before_launch(pkg):
    L, E, N = pkg.lib(), pkg.ERROR_INVALID_VALUE, pkg.ERROR_NOT_SUPPORTED
    good = cache_of(pkg)
    for over in BAD_CACHES:
        c = cache_of(pkg, **over)
        assert L.iq4xs_qk_norm_rope_append(qk_args(pkg), c, None) == E, over
        assert L.iq4xs_kv_gather(c, FAKE, 2, FAKE, 1, FAKE, FAKE, 4, 1, None) == E, over
        assert L.iq4xs_paged_attention(attention_args(pkg, c), None, 0, None) == E, over
    odd = cache_of(pkg, d=96)
    assert L.iq4xs_kv_gather(odd, FAKE, 2, FAKE, 1, FAKE, FAKE, 4, 1, None) == N
    assert L.iq4xs_paged_attention(attention_args(pkg, odd), None, 0, None) == N
    for over in BAD_QK:
        assert L.iq4xs_qk_norm_rope(qk_args(pkg, **over), None) == E, over
        assert L.iq4xs_qk_norm_rope_append(qk_args(pkg, **over), good, None) == E, over
    assert L.iq4xs_qk_norm_rope(qk_args(pkg, ko=0), None) == E
    assert L.iq4xs_qk_norm_rope(qk_args(pkg, d=96, qs=384, ks=192, rot=96), None) == N
    assert L.iq4xs_qk_norm_rope(qk_args(pkg, rot=24), None) == N
    for over in (dict(v=0), dict(slots=0), dict(vs=128), dict(hk=3, ks=384, vs=384), dict(d=64, rot=64)):
        assert L.iq4xs_qk_norm_rope_append(qk_args(pkg, **over), good, None) == E, over
    assert L.iq4xs_qk_norm_rope(None, None) == E and L.iq4xs_qk_norm_rope_append(qk_args(pkg), None, None) == E
    for a in ((None, 2, FAKE, 1, FAKE, FAKE, 4, 1), (FAKE, 0, FAKE, 1, FAKE, FAKE, 4, 1),
              (FAKE, 2, None, 1, FAKE, FAKE, 4, 1), (FAKE, 2, FAKE, -1, FAKE, FAKE, 4, 1),
              (FAKE, 2, FAKE, 1, None, FAKE, 4, 1), (FAKE, 2, FAKE, 1, FAKE, FAKE + 8, 4, 1),
              (FAKE, 2, FAKE, 1, FAKE, FAKE, -1, 1), (FAKE, 2, FAKE, 1, FAKE, FAKE, 4, 3)):
        assert L.iq4xs_kv_gather(good, *a, None) == E, a
    for over in BAD_ATTENTION:
        args = attention_args(pkg, good, **over)
        assert L.iq4xs_paged_attention_workspace_bytes(args) == 0, over
        assert L.iq4xs_paged_attention(args, FAKE, 1 << 40, None) == E, over
    assert L.iq4xs_paged_attention(None, None, 0, None) == E


def test_nothing_to_do_launches_nothing(pkg):
    L, good = pkg.lib(), cache_of(pkg)
    assert L.iq4xs_qk_norm_rope(qk_args(pkg, tokens=0, q=0), None) == 0
    assert L.iq4xs_qk_norm_rope_append(qk_args(pkg, tokens=0), good, None) == 0
    assert L.iq4xs_kv_gather(good, FAKE, 2, FAKE, 1, FAKE, FAKE, 0, 1, None) == 0
    for over in (dict(total=0), dict(seqs=0)):
        args = attention_args(pkg, good, **over)
        assert L.iq4xs_paged_attention_workspace_bytes(args) == 0
        assert L.iq4xs_paged_attention(args, None, 0, None) == 0
