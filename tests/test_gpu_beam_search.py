"""The serving operators together: beam search over forked 4-bit histories, and the same tokens scored as one prompt.

A beam's score is the sum of log probabilities found while its history was forked, grown and copied from page to page;
prefilling prompt and tokens into a fresh cache has to give the same sum. The two differ only where attention's last
float32 bits move an int8 activation across a rounding: one step in 127 of a block's largest value, in a sum of at least
64 such products -- 1e-2 for each token is several of those, and a wrong page changes logits by tenths.
"""

from __future__ import annotations

import numpy as np
import pytest

from examples.beam_search import Decoder, beam_search, prefill
from nanocompile_b200 import model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams,tokens,prompt_length", [(1, 5, 3), (4, 20, 37), (7, 33, 16)])
def test_beams_score_what_their_tokens_score_as_a_prompt(cuda, beams, tokens, prompt_length):
    shape = model.SMALL
    weights = model.synthetic_weights(shape, seed=3, std=0.08)
    prompt = model.synthetic_prompt(shape.vocab, prompt_length)
    decoder = Decoder(shape, weights, beams, prompt_length + tokens)
    found = beam_search(decoder, prompt, tokens)
    assert len(found) == beams and [b.score for b in found] == sorted((b.score for b in found), reverse=True)
    assert len({tuple(b.tokens) for b in found}) == beams
    single = Decoder(shape, weights, 1, prompt_length + tokens)
    for beam in found:
        assert len(beam.tokens) == tokens
        ids = prompt + beam.tokens
        prefill(single, ids[:-1], targets=ids[1:])
        logprobs = single.logprobs.numpy()[prompt_length - 1:, 0]
        assert abs(float(logprobs.astype(np.float64).sum()) - beam.score) <= 1e-2 * tokens


def test_one_beam_takes_the_best_token_each_time(cuda):
    shape = model.SMALL
    weights = model.synthetic_weights(shape, seed=5, std=0.08)
    prompt = model.synthetic_prompt(shape.vocab, 20)
    beam = beam_search(Decoder(shape, weights, 1, 40), prompt, 12)[0]
    single = Decoder(shape, weights, 1, 40)
    ids = prompt + beam.tokens
    prefill(single, ids[:-1], targets=ids[1:])
    best, given = single.top_logprobs.numpy()[19:, 0], single.logprobs.numpy()[19:, 0]
    assert (best - given <= 1e-2).all()
