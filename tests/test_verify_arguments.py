"""What the wrapper of the verification hands to the library: rows longer than the vocabulary, on the CPU."""
import pytest

from ingot_amd import Session
from ingot_amd import _lib as L
from ingot_amd.host import DeviceTensor


def tensor(dtype, *shape):
    return DeviceTensor(None, dtype, shape, 4096, False)


@pytest.fixture
def verify():
    s = Session.__new__(Session)
    s.lib, s.h = L.load(), None
    s._prepared = lambda fn, *a: a
    out = tensor(L.DT_I32, 2, 4), tensor(L.DT_I32, 2), tensor(L.DT_I32, 2)

    def of(logits, **kw):
        args = s.prepare_verify_drafts(logits, tensor(L.DT_I32, 3), tensor(L.DT_I32, 3), *out, **kw)[0]._obj
        return args.vocab, args.logits_ld, args.draft_ld, args.tokens

    return of


def test_rows_longer_than_the_vocabulary(verify):
    assert verify(tensor(L.DT_F32, 3, 9))[:2] == (9, 9)
    assert verify(tensor(L.DT_F32, 3, 16), vocab=9)[:2] == (9, 16)
    assert verify(tensor(L.DT_F32, 3, 16), vocab=9, draft=tensor(L.DT_F32, 3, 9)) == (9, 16, 9, 3)
    assert verify(tensor(L.DT_F32, 3, 9), vocab=9, draft=tensor(L.DT_F32, 3, 32)) == (9, 9, 32, 3)


def test_refusals(verify):
    logits = tensor(L.DT_F32, 3, 9)
    for kw in (dict(vocab=10), dict(vocab=9, draft=tensor(L.DT_F32, 3, 8)), dict(vocab=8, draft=tensor(L.DT_F32, 4, 9)),
               dict(vocab=8, draft=tensor(L.DT_BF16, 3, 9)), dict(vocab=8, draft=tensor(L.DT_F32, 27)),
               dict(draft=tensor(L.DT_F32, 3, 10))):
        with pytest.raises(ValueError, match="verify_drafts"):
            verify(logits, **kw)
