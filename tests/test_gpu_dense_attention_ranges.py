"""dense_attention over the whole range of its arguments: values that are not finite, distances that count for a key, scales and caps at both
ends, fp16 gradients of small size.  Bounds: tests/dense_reference.py."""
import math

import pytest
import torch

from tests import dense_reference as R
from tests.test_gpu_dense_attention import _dense, _inputs

pytestmark = pytest.mark.gpu


# ---- values that are not finite where nothing sees them ----------------------------------------------------------------------------

@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_documents_keep_their_gradients_apart(cap, poison, D, dtype):
    """q, k, v and dout of the rows before the first document and behind the last, and of a whole document in between, hold NaN or infinities:
    outputs and gradients of the documents beside them stay within their bounds, the gradients of rows of no document are zero."""
    S, cu = 420, [20, 150, 290, 400]
    q, k, v, dout = _inputs(1, 4, 2, S, S, D, dtype, seed=20)
    lo, hi, pos = R.runs(1, S, S, True, [(cu, cu)], None, None)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), cap, None, dout)
    for x in (q, k, v, dout):
        x[:, :, :20] = x[:, :, 400:] = x[:, :, 150:290] = poison
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, causal=True, softcap=cap, cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    grads = torch.autograd.grad(out, leaves, dout)
    rows = [*range(20, 150), *range(290, 400)]
    outside = [*range(20), *range(400, S)]
    for got, x in zip((out.detach(), *grads), ("o", "dq", "dk", "dv")):
        val, bound = want[x]
        assert R.worst(got[:, :, rows], (val[:, :, rows], bound[:, :, rows])) <= 1, x
        assert not got[:, :, outside].any(), x
