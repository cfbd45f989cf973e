"""Edges of what the serving operators take, without a GPU: a block of zeros stands for the handle and numbers for the addresses (every refusal comes
before the device is touched; a call that is fine but for its workspace says how large that has to be)."""
import pytest

from test_serving_refusals import A, call, scores


@pytest.mark.parametrize("ty,size", [(0, 4), (1, 2), (30, 2)])
def test_the_largest_vocabulary(ty, size):
    """A row's last turn (512 f32, 1024 16-bit values) and piece end below 2^31 wherever the row starts."""
    def row(vocab):
        return scores(type=ty, rows=1, top=0, vocab=vocab, logits=A[11], stride=vocab * size, tokens=0, logprob=A[2], entropy=0, top_ids=0, top_logprobs=0, workspace_bytes=0)
    call("tlb_token_logprobs", row(2 ** 31 - 2048), "workspace of", "Invalid")
    for vocab in (2 ** 31 - 2047, 2 ** 31 - 1024, 2 ** 31 - 257, 2 ** 31):
        call("tlb_token_logprobs", row(vocab), "tokens", "Unsupported")
