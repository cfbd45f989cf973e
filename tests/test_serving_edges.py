"""Edges of what the serving operators take, without a GPU: a block of zeros stands for the handle and numbers for the addresses (every refusal comes
before the device is touched; a call that is fine but for its workspace says how large that has to be)."""
import pytest

from test_serving_refusals import A, call, keep, scores


@pytest.mark.parametrize("ty,size", [(0, 4), (1, 2), (30, 2)])
def test_the_largest_vocabulary(ty, size):
    """A row's last turn (512 f32, 1024 16-bit values) and piece end below 2^31 wherever the row starts."""
    def row(vocab):
        return scores(type=ty, rows=1, top=0, vocab=vocab, logits=A[11], stride=vocab * size, tokens=0, logprob=A[2], entropy=0, top_ids=0, top_logprobs=0, workspace_bytes=0)
    call("tlb_token_logprobs", row(2 ** 31 - 2048), "workspace of", "Invalid")
    for vocab in (2 ** 31 - 2047, 2 ** 31 - 1024, 2 ** 31 - 257, 2 ** 31):
        call("tlb_token_logprobs", row(vocab), "tokens", "Unsupported")


# ------------------------------------------------------------------------------------------------ what shares a byte and what lies between
@pytest.mark.parametrize("change", [dict(logprob=A[0] + 400), dict(entropy=A[0] + 512 + 484), dict(top_ids=A[0] + 400), dict(tokens=A[0] + 496)])
def test_results_between_strided_logits_are_fine(change):
    """Rows of 400 bytes, 512 apart; the refusal that follows is another one."""
    call("tlb_token_logprobs", scores(stride=512, workspace_bytes=16, **change), "workspace of", "Invalid")


@pytest.mark.parametrize("change", [
    dict(logprob=A[0] + 396), dict(entropy=A[0] + 508), dict(top_ids=A[0] + 468), dict(top_logprobs=A[0] + 1024 - 16), dict(status=A[0] + 1024 + 200), dict(logprob=A[0] - 8),
    dict(workspace=A[0] + 464)])
def test_results_on_strided_logits_are_refused(change):
    call("tlb_token_logprobs", scores(stride=512, **change), "overlaps", "Invalid")


def test_pools_of_layers_in_turn():
    pool = 20 * 2 * 16 * 64 * 2
    for fine in (dict(v_pools=A[0] + pool), dict(k_pools=A[0] + pool, v_pools=A[0]), dict(v_pools=A[0] + pool, v_layer_stride=2 * pool, layers=1, k_layer_stride=0),
                 dict(v_pools=A[0] + 5 * pool), dict(v_pools=A[0] + 3 * pool, k_layer_stride=pool, v_layer_stride=pool)):
        call("tlb_cache_keep", keep(tables=A[4] + 2, **fine), "4-byte", "Invalid")
    for bad in (dict(v_pools=A[0] + pool - 16), dict(v_pools=A[0] + 2 * pool + 16), dict(v_pools=A[0] + pool, v_layer_stride=3 * pool), dict(v_pools=A[0] + 2 * pool, k_layer_stride=pool, v_layer_stride=pool)):
        call("tlb_cache_keep", keep(**bad), "overlap", "Invalid")


def test_numbers_inside_the_pools_are_refused():
    """What cache_keep moves could overwrite the tables and paths that say where to."""
    pool = 20 * 2 * 16 * 64 * 2
    for name in ("tables", "context", "counts", "path", "status"):
        for at in (A[0] + 64, A[0] + pool + 4096, A[0] + 6 * pool - 4):
            call("tlb_cache_keep", keep(**{name: at}), "overlap", "Invalid")
    call("tlb_cache_keep", keep(status=A[4] + 8), "overlap", "Invalid")
    # between the layers there is room
    call("tlb_cache_keep", keep(k_layer_stride=4 * pool, v_layer_stride=4 * pool, context=A[0] + 2 * pool, counts=A[0] + 4 * pool - 8, tables=A[4] + 2), "4-byte", "Invalid")
