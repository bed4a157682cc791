"""What the preparation of a chunk leaves for the scan: lower triangles with zeros above, whatever the workspace held before."""
import pytest
import torch

from .test_hybrid_passes_gpu import D, _Call

pytestmark = pytest.mark.gpu
KEY_BYTES, TRI, HEAD_BYTES, UNITS = 4 * 64 * D * 2, 64 * 64 * 2, 4 * 64 * 64 * 2 + 64 * D * 4 + 4 * 64 * 4, 3


def _workspace(monkeypatch, fill):
    from llaminar_b200.ops import hybrid
    one, held = hybrid.ext().gdn_chunk_bytes(1, 16, 16), []
    assert one == 16 * (KEY_BYTES + HEAD_BYTES)

    def workspace(inp, *_):
        held.append(torch.full((UNITS * one + 1024,), fill, dtype=torch.uint8, device=inp.device))
        return held[-1]

    monkeypatch.setattr(hybrid, "_gdn_workspace", workspace)
    return held


@pytest.mark.parametrize("lens,pos", [([140], [0]), ([64, 37], [5, 0])])
def test_triangles_have_zeros_above_and_results_do_not_depend_on_the_workspace(monkeypatch, lens, pos):
    """The scan multiplies whole 64 x 64 triangles: products of one shape, whose order is promised."""
    results = []
    for fill in (0, 255):
        held = _workspace(monkeypatch, fill)
        call = _Call(lens, pos)
        call.run()
        results.append(call.results())
    for a, b in zip(*results):
        assert torch.equal(a, b)
    ws = held[0]
    ws = ws[-ws.data_ptr() % 1024:]
    heads = ws[UNITS * 16 * KEY_BYTES:][:UNITS * 16 * HEAD_BYTES].view(UNITS, 16, HEAD_BYTES)
    used = sum(-(-n // 64) for n in lens)
    images = heads[:used, :, :4 * TRI].reshape(used * 16, 4, 64, 8, 16)             # T and P as two numbers each, rows of eight 16-byte units
    t, u = torch.meshgrid(torch.arange(64), torch.arange(8), indexing="ij")
    images = images[:, :, t, u ^ (t & 7)].contiguous().view(torch.float16).reshape(-1, 4, 64, 64)        # (a unit lies where its row's low bits put it)
    assert (images.triu(1) == 0).all() and torch.isfinite(images.float()).all()
    assert (images[:, 0].diagonal(dim1=1, dim2=2) == 4096).all()                    # T has ones on the diagonal, times 2^12
