"""Beams of several requests with adapters of their own, chosen on the device: the operators together, as a server would run them.

A beam's score, summed up by the choices while its history was forked, moved and cut, has to be what its tokens score as one prompt
with the request's adapter in a fresh cache. The two differ only where attention's or an adapter's last float32 bits move an int8
activation across a rounding: the bound of ``test_gpu_beam_search``, 1e-2 a token.
"""

from __future__ import annotations

import numpy as np
import pytest

from examples.beam_search import Adapters, Decoder, beam_search, beam_search_requests, prefill
from nanocompile_b200 import model

pytestmark = pytest.mark.gpu


def rescored(decoder, prompt, tokens, adapter):
    if decoder.adapters:
        decoder.use([adapter])
    ids = list(prompt) + tokens
    prefill(decoder, ids[:-1], targets=ids[1:])
    return float(decoder.logprobs.numpy()[len(prompt) - 1:, 0].astype(np.float64).sum())


@pytest.mark.parametrize("beams,tokens,end", [(1, 6, -1), (4, 20, 5), (5, 17, -1)])
def test_beams_of_requests_score_what_their_tokens_score_as_a_prompt(cuda, beams, tokens, end):
    shape = model.SMALL
    weights, adapters = model.synthetic_weights(shape, seed=3, std=0.08), Adapters(shape, slots=4, rank=16, seed=1)
    prompts = [model.synthetic_prompt(shape.vocab, n) for n in (21, 1, 34)]
    ids = [2, -1, 0]
    decoder = Decoder(shape, weights, beams * 3, 34 + tokens, adapters=adapters)
    found = beam_search_requests(decoder, prompts, beams, tokens, ids, end)
    single = Decoder(shape, weights, 1, 34 + tokens, adapters=adapters)
    for prompt, adapter, best in zip(prompts, ids, found):
        assert [b.score for b in best] == sorted((b.score for b in best), reverse=True)
        assert len({tuple(b.tokens) for b in best}) == beams
        for beam in best:
            assert len(beam.tokens) == tokens or beam.tokens[-1] == end
            assert end not in beam.tokens[:-1]
            assert abs(rescored(single, prompt, beam.tokens, adapter) - beam.score) <= 1e-2 * len(beam.tokens)


def test_one_request_finds_what_the_host_finds(cuda):
    """Without adapters, the device's choice and the host's: the same beams, but for totals that lie as close as their float32 sums."""
    shape = model.SMALL
    weights, prompt = model.synthetic_weights(shape, seed=3, std=0.08), model.synthetic_prompt(shape.vocab, 37)
    host = beam_search(Decoder(shape, weights, 4, 60), prompt, 12)
    device = beam_search_requests(Decoder(shape, weights, 4, 60), [prompt], 4, 12)[0]
    for a, b in zip(host, device):
        assert a.tokens == b.tokens or abs(a.score - b.score) <= 12 * 4e-6
        assert abs(a.score - b.score) <= 12 * 4e-6


def test_an_adapter_changes_its_requests_alone(cuda):
    """A batch's requests with an adapter and without: the ones without find what they find alone."""
    shape = model.SMALL
    weights, adapters = model.synthetic_weights(shape, seed=5, std=0.08), Adapters(shape, slots=2, rank=8, seed=2)
    prompt = model.synthetic_prompt(shape.vocab, 12)
    both = beam_search_requests(Decoder(shape, weights, 4, 30, adapters=adapters), [prompt, prompt], 2, 8, [-1, 1])
    alone = beam_search_requests(Decoder(shape, weights, 2, 30), [prompt], 2, 8)[0]
    assert [b.tokens for b in both[0]] == [b.tokens for b in alone]
    assert [b.score for b in both[0]] != [b.score for b in both[1]]
