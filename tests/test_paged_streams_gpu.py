"""A paged cache's calls on a stream that is asked for, with inputs that have to be copied: the copies are that stream's work, whatever the current one is busy with.  And
angles of one position, whose stride may be any."""
import pytest
import torch

from paged_cases import FP8, Cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def busy():
    """Some hundred milliseconds of work for the current stream."""
    x = torch.zeros(8192, 8192, dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    for _ in range(200):
        x = x @ x


def turned_round(t):
    """The same values, the innermost dimension not next to each other."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


def every_other(t):
    return torch.stack([t, t], -1)[..., 0]


@pytest.mark.parametrize("as_handle", [False, True])
@pytest.mark.parametrize("held", [torch.float16, FP8])
def test_attend(ops, held, as_handle):
    cache = Cache([300, 1, 77, 0], 2, 16, 64, held)
    table, n = cache.tensors(DEV)
    c, q = cache.on(ops, DEV), torch.randn(4, 8, 64).half().to(DEV)
    want = c.attend(q, table, n, lse=True)
    qs, ts, ns = turned_round(q), turned_round(table), every_other(n)
    assert qs.stride(2) != 1 and ts.stride(1) != 1 and ns.stride(0) != 1
    s = torch.cuda.Stream()
    busy()
    got = c.attend(qs, ts, ns, lse=True, stream=s.cuda_stream if as_handle else s)
    s.synchronize()
    assert not torch.cuda.current_stream().query()   # (else the current stream's work was done before, and this has shown nothing)
    with torch.cuda.stream(s):
        got = [t.cpu() for t in got]
    assert all(torch.equal(a, b.cpu()) for a, b in zip(got, want))
    torch.cuda.synchronize()


@pytest.mark.parametrize("as_handle", [False, True])
@pytest.mark.parametrize("held", [torch.float16, FP8])
def test_append(ops, held, as_handle):
    cache = Cache([40, 5, 17], 2, 16, 64, held)
    table, n = cache.tensors(DEV)
    a, b = cache.on(ops, DEV), cache.on(ops, DEV)
    starts = torch.tensor([0, 20, 21, 30], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(30, h, 64, generator=g).half().to(DEV) for h in (4, 2, 2))
    angles = ops.rotary_table(table.size(1) * 16, 64, device=DEV)
    want = a.append(k, v, table, n, starts=starts, q=q, rotary=angles)
    args = turned_round(k), turned_round(v), turned_round(table), every_other(n)
    more = dict(starts=every_other(starts), q=turned_round(q), rotary=turned_round(angles))
    s = torch.cuda.Stream()
    busy()
    got = b.append(*args, **more, stream=s.cuda_stream if as_handle else s)
    s.synchronize()
    assert not torch.cuda.current_stream().query()
    raw = torch.uint8 if held == FP8 else torch.int16
    with torch.cuda.stream(s):
        got, pages = got.cpu(), [t.view(raw).cpu() for t in (b.k_pages, b.v_pages)]
    assert torch.equal(got, want.cpu())
    assert all(torch.equal(x, y.view(raw).cpu()) for x, y in zip(pages, (a.k_pages, a.v_pages)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("stride", [1, 3, 16, 40])
def test_angles_of_one_position(ops, stride):
    """A cache with room for one token: its angles are one row."""
    k = torch.randn(2, 1, 16).half().to(DEV)
    table, n = torch.tensor([[1], [0]], dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    c, d = (ops.PagedCache(*(torch.zeros(2, 1, 1, 16, dtype=torch.float16, device=DEV) for _ in range(2))) for _ in range(2))
    angles = torch.rand(16, device=DEV)
    want = c.append(k, k, table, n, q=k, rotary=angles.view(1, 16))
    one = torch.cat([angles, torch.zeros(40, device=DEV)]).as_strided((1, 16), (stride, 1))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = d.append(k, k, table, n, q=k, rotary=one, stream=s)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(c.k_pages, d.k_pages)
