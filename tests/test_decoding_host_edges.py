"""Calls around the quantised cache at the edges of what is documented: nothing to do, one page, the caller's own tensors.  No GPU."""
import pytest

pytest.importorskip("torch")

from attention_reference import load_abq_attention  # noqa: E402
from test_decoding_host import ref, sparse  # noqa: E402
from test_attention_host import A  # noqa: E402


@pytest.fixture(scope="module")
def attn():
    return load_abq_attention()


def test_attention_to_chosen_pages_without_drafts(attn):
    """No rows: there is nothing to list pages for, and an empty tensor has no address"""
    L, ok = attn.lib(), attn.abq_gemm
    none = {"rows": 0, "data": None}
    s, st = sparse(attn, q=none, out=none, blocks=None)
    assert s == ok.ABQ_OK and L.abq_attn_sparse_exec(ref(st), None) == ok.ABQ_OK
    assert L.abq_attn_sparse_workspace_bytes(ref(st)) == 0 and L.abq_attn_sparse_set_workspace(ref(st), None, 0) == ok.ABQ_OK
    for kw in ({"count": 0}, {"blocks": None}, {"blocks": None, "q": {"rows": 0}}):
        assert sparse(attn, **kw)[0] == ok.ABQ_ERR_INVALID_ARG, kw
    assert sparse(attn, blocks=A)[0] == ok.ABQ_OK
