"""Adapted rows and queries on their way into an index on one stream, without a wait in between, and
adapter calls captured behind work of another stream."""
import numpy as np
import pytest
import torch

from adapter_cases import Maker, ptr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


@pytest.mark.parametrize("storage", ["fp32", "fp16"])
def test_adapted_rows_are_added_and_adapted_queries_search_them(oracle, xb, storage):
    """Both sides of a two-tower search: rows through one layer into add_device, queries through a gated
    block and a layer into search_device; equal to the oracle on the adapted vectors."""
    n, rows, k, m = 37, 2500, 96, 64
    mk = Maker(storage, 3)
    x, base = mk.matrix(n, k).contiguous(), mk.matrix(rows, k).contiguous()
    w, wg, wu, wd = (mk.matrix(*s, k ** -0.5).contiguous() for s in ((m, k), (m, k), (m, k), (m, m)))
    kind = xb.STORAGE_FP32 if storage == "fp32" else xb.STORAGE_FP16
    new = lambda *s: torch.empty(s, device="cuda", dtype=x.dtype)
    adapted, h, q = new(rows, m), new(n, m), new(n, m)
    keys = torch.arange(rows, device="cuda", dtype=torch.int64) * 3 + 1
    okeys = torch.zeros(n, 10, dtype=torch.int64, device="cuda")
    oscores = torch.zeros(n, 10, device="cuda")
    ocounts = torch.zeros(n, dtype=torch.int32, device="cuda")
    idx = xb.DenseFlatIndex(m, xb.METRIC_COSINE, storage=kind)
    s = torch.cuda.current_stream().cuda_stream
    xb.linear_device(0, kind, rows, k, m, ptr(base), ptr(w), ptr(adapted), activation=xb.ACT_GELU, stream=s)
    idx.add_device(ptr(keys), ptr(adapted), rows, stream=s)
    xb.gated_device(0, kind, n, k, m, ptr(x), ptr(wg), ptr(wu), ptr(h), stream=s)
    xb.linear_device(0, kind, n, m, m, ptr(h), ptr(wd), ptr(q), residual_ptr=ptr(h), stream=s)
    idx.search_device(ptr(q), n, xb.SearchOptions(top_k=10), ptr(okeys), ptr(oscores), ptr(ocounts), stream=s)
    torch.cuda.synchronize()
    st, want, scores, counts, _ = oracle.flat_search(
        xb.METRIC_COSINE, adapted.float().cpu().numpy(), keys.cpu().numpy().astype(np.uint64),
        q.float().cpu().numpy(), 10)
    assert st == 0 and np.array_equal(ocounts.cpu().numpy(), counts)
    assert np.array_equal(okeys.cpu().numpy().astype(np.uint64), want)
    assert np.array_equal(oscores.cpu().numpy().view(np.uint32), scores.view(np.uint32))
    idx.close()


@pytest.mark.parametrize("n", [2, 200])
@pytest.mark.parametrize("kind", ["fp32", "fp16"])
def test_captured_behind_another_streams_work(xb, n, kind):
    """A captured call whose input comes from another stream, joined by an event after a long kernel
    there: its early launch still waits for both streams."""
    k = m = 256
    mk = Maker(kind, 4)
    storage = 1 if kind == "fp32" else 2
    x, w = mk.matrix(n, k).contiguous(), mk.matrix(m, k, k ** -0.5).contiguous()
    late = torch.zeros_like(x)
    first, y = (torch.empty(n, m, device="cuda", dtype=x.dtype) for _ in range(2))
    big = torch.randn(6000, 6000, device="cuda")
    room = torch.empty_like(big)

    def step():
        s, other = torch.cuda.current_stream(), torch.cuda.Stream()
        xb.linear_device(0, storage, n, k, m, ptr(x), ptr(w), ptr(first), stream=s.cuda_stream)
        other.wait_stream(s)
        with torch.cuda.stream(other):
            torch.matmul(big, big, out=room)
            late.copy_(x)
        s.wait_stream(other)
        xb.linear_device(0, storage, n, k, m, ptr(late), ptr(w), ptr(y), stream=s.cuda_stream)
        late.zero_()

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, first)
    del graph
