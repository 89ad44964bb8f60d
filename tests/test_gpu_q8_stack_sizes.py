"""GPU: the hybrid stack with its feed-forward in 8-bit integers at the served width of the feed-forward, and at one above 4096, whose steps go another way."""
import pytest

import test_gpu_q8_stack as small

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[3584, 4352])
def wide(request, monkeypatch):
    monkeypatch.setattr(small, "INTER", request.param)


@pytest.mark.parametrize("seqs,tokens,chunk", [(1, 1, 1), (1, 16, 1), (3, 7, 3), (2, 300, 2)])
def test_prompts(ops, cuda, synth, wide, seqs, tokens, chunk):
    small.test_prompts(ops, cuda, synth, seqs, tokens, chunk)


@pytest.mark.parametrize("rows,gemm", [(1, ""), (2, ""), (8, ""), (16, ""), (17, ""), (128, ""), (3, "tc"), (3, "cublas")])
def test_decode_steps(ops, cuda, synth, monkeypatch, wide, rows, gemm):
    small.test_decode_steps(ops, cuda, synth, monkeypatch, rows, gemm)


def test_single_tokens_give_the_logits_of_the_rows(ops, cuda, synth, wide):
    small.test_single_tokens_give_the_logits_of_the_rows(ops, cuda, synth)
