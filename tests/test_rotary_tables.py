"""The rotation tables that an attention module keeps: for what it is now, and none of a saved module's."""
import copy
import io

import pytest
import torch

from oracle import kv8 as ref


def _module(**kw):
    from energonai_amd.model import MultiHeadAttention1D
    return MultiHeadAttention1D(**{**dict(hidden_size=64, num_heads=2, max_seq_len=16, rotary_dim=32), **kw})


CPU = torch.device("cpu")


def test_tables_follow_the_module():
    m = _module()
    assert m._rotary(CPU, 16)[0].shape == (16, 16) and m._rotary(CPU, 16)[0] is m._rotary(CPU, 3)[0]
    with pytest.raises(RuntimeError):
        m._rotary(CPU, 17)
    first = m._rotary(CPU, 16)
    m.max_seq_len = 64
    cos, sin = m._rotary(CPU, 40)
    want = ref.table(64, 32)
    assert cos.shape == (64, 16) and torch.allclose(cos, want[0], atol=1e-6) and torch.allclose(sin, want[1], atol=1e-6)
    m.rotary_base = 500.0
    assert torch.allclose(m._rotary(CPU, 40)[1], ref.table(64, 32, 500.0)[1], atol=1e-6)
    m.rotary_dim = 8
    assert m._rotary(CPU, 40)[0].shape == (64, 4)
    m.kv_page_size = 128
    assert m._rotary(CPU, 40)[0].shape == (128, 4)
    # and back: a captured step goes on reading the tables it was captured with
    m.max_seq_len, m.rotary_base, m.rotary_dim, m.kv_page_size = 16, 10000.0, 32, None
    assert m._rotary(CPU, 16)[0] is first[0]
    m.rotary_dim = 0
    assert m._rotary(CPU, 40) is None


def test_turned_follows_the_module():
    m = _module(rotary_dim=0)
    assert not m.turned
    m.rotary_dim = 32
    assert m.turned and _module(rotary_dim=0, qk_norm=True).turned


def test_tables_are_not_saved():
    m = _module()
    m._rotary(CPU, 16)
    for other in (copy.deepcopy(m), copy.copy(m)):
        assert not other._rotary_tables
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    # tensors of `cpu` that come back elsewhere, as those of a GPU do that come back on the CPU
    back = torch.load(f, map_location="meta", weights_only=False)
    assert back._rotary(CPU, 16)[0].device == CPU and back.query_key_value.weight.device.type == "meta"
    assert m._rotary_tables                                       # those of the module itself stay


def test_a_module_saved_with_tables():
    """One whose state has tables in it, keyed by a device that they are no longer on."""
    m = _module()
    state = dict(m.__dict__, _rotary_tables={CPU: tuple(torch.empty(16, 16, device="meta") for _ in range(2))}, turned=True)
    back = type(m).__new__(type(m))
    back.__setstate__(state)
    assert back._rotary(CPU, 16)[0].device == CPU and back.turned


def test_the_step_has_tables_for_its_cache():
    """A cache that was started under a larger max_seq_len goes on to its end."""
    m = _module(is_decoder=True)
    seen = []

    class Cache:
        max_seq_len = 48

        def append_rotary(self, q, k, v, rotary, **how):
            seen.append(rotary[0].shape)
            return q

        def attend(self, q, scale):
            return q[:, :, None]
    m.kv_cache = Cache()
    m.float()
    m.forward_last(torch.zeros(1, 1, 64))
    assert seen == [(48, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(kv_page_size=16), dict(kv_cache_dtype=torch.int8)])
def test_a_used_module_goes_on(kw):
    """A module that has run takes longer prompts once max_seq_len is raised, and runs again after a trip to the CPU in a file: as a new one does."""
    from energonai_amd.model import MultiHeadAttention1D
    from gpu_util import announce
    announce("rotary tables of a used module", kw)
    make = lambda n: MultiHeadAttention1D(64, 2, dtype=torch.float16, max_seq_len=n, rotary_dim=32, qk_norm=True, **kw)  # noqa: E731
    m, new = make(32).cuda().eval(), make(128).cuda().eval()
    new.load_state_dict(m.state_dict())
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn(2, n, 64, generator=g).half().cuda() for n in (20, 100))
    last = torch.randn(2, 1, 64, generator=g).half().cuda()
    lens = torch.tensor([100, 77], dtype=torch.int32).cuda()
    with torch.no_grad():
        m(x, first_cache=True, seq_lens=torch.tensor([20, 3], dtype=torch.int32).cuda())
        m.max_seq_len = 128
        m.kv_cache = None
        f = io.BytesIO()
        torch.save(m, f)
        f.seek(0)
        back = torch.load(f, map_location="cpu", weights_only=False).cuda()
        want = [new(y, first_cache=True, seq_lens=lens)] + [new(last) for _ in range(18)]
        for other in (m, back):
            got = [other(y, first_cache=True, seq_lens=lens)] + [other(last) for _ in range(18)]
            assert all(bool(torch.isfinite(t).all()) for t in got) and all(torch.equal(a, b) for a, b in zip(got, want))
