"""Arguments of the 4-bit attention that are kept or handed on by the binding."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def test_the_workspace_is_asked_for_per_type(torch, monkeypatch):
    """The launch's shape is found by the occupancy of the type's own kernel: what one type needs is not what another does."""
    from agxforge.kernels import kv4
    from agxforge_b200 import _native as N
    L = N.lib()
    asked = []
    ask = L.agxc_kv4_attention_workspace

    class Lib:
        def __getattr__(self, name):
            if name != "agxc_kv4_attention_workspace":
                return getattr(L, name)
            return lambda ctx, a: (asked.append(a._obj.dtype), ask(ctx, a))[1]

    monkeypatch.setattr(N, "lib", lambda: Lib())
    c = kv4.KV4Cache(2, 2, 64, 16)
    table, lens = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for dtype in (torch.float16, torch.bfloat16) * 2:
        kv4.attention(torch.zeros((1, 4, 64), dtype=dtype, device="cuda"), c, table, lens)
    assert sorted(asked) == [N.F16, N.BF16]
    # a server's page tables have every width: what is remembered stays small
    for rows in range(1, 3000):
        c._workspace[("shape", rows)] = 0
    kv4.attention(torch.zeros((1, 3, 4, 64), dtype=torch.float16, device="cuda"), c, table, lens)
    assert len(c._workspace) <= 1024


def test_a_page_tables_stride_past_32_bits(torch):
    """Rows further apart than the call can say are refused, not taken from elsewhere."""
    from agxforge.kernels import kv4
    c = kv4.KV4Cache(2, 2, 64, 16)
    store = torch.zeros((1 << 32) + 8, dtype=torch.int32, device="cuda")
    q, lens = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for stride in (1 << 31, (1 << 32) + 2):
        with pytest.raises(ValueError, match="page_table"):
            kv4.attention(q, c, store.as_strided((2, 2), (stride, 1)), lens)
    kv4.attention(q, c, store.as_strided((2, 2), (1000, 1)), lens)
