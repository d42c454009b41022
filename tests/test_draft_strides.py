"""Row strides that the library's int32 does not hold are refused, not cut off."""
import pytest
import torch

from ferrisinfer_amd import FerrisError
from test_draft_refusals import CALLS, context


@pytest.mark.parametrize("what", ["logits", "draft_probs"])
@pytest.mark.parametrize("stride,kind", [(2 ** 31 - 1, "InvalidConfig"), (2 ** 31, "Unsupported"), (2 ** 32 + 64, "Unsupported"),
                                         (2 ** 33, "Unsupported")])
def test_rows_far_apart(what, stride, kind):
    far = torch.empty_strided((6, 50), (stride, 1), device="meta")
    with pytest.raises(FerrisError) as e:
        context().verify_drafts(**dict(CALLS["verify_drafts"], **{what: far}))
    assert e.value.kind == kind and (kind == "InvalidConfig" or what in e.value.message)  # (InvalidConfig: it reached the library)


def test_one_row_has_no_stride():
    one = dict(CALLS["verify_drafts"], logits=torch.empty_strided((1, 50), (2 ** 40, 1), device="meta"), draft_probs=None)
    with pytest.raises(FerrisError) as e:
        context().verify_drafts(**one)
    assert e.value.kind == "InvalidConfig"
