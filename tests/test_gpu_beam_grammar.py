"""Beams under a grammar: ByteDfa.mask's bits are beam_select's, the beams'
automaton states follow their parents."""
import re

import numpy as np
import pytest
import torch

from tests.test_gpu_beam import _ctx, beams, check, empty_pool, rows_at

pytestmark = pytest.mark.gpu

PATTERN = "(ab|cd|a)+(e|fgh)?"


def grammar():
    from zllm_amd.engine import LogitFSM, TokenByteTable
    tokens = [bytes([b]) for b in b"abcdefgh"] + [b"ab", b"cda", b"bcd", b"fg", None, b"gh"]
    eos = len(tokens)
    table = TokenByteTable(_ctx(), tokens + [b""], eos)
    return LogitFSM.compile("regex:" + PATTERN, table), table, tokens, eos


def unpacked(bits, V):
    return np.unpackbits(bits.cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)


def test_a_search_stays_in_its_grammar():
    from zllm_amd.beam import BeamSearch, BeamStates, beam_reorder
    fsm, table, tokens, eos = grammar()
    rng = np.random.default_rng(2)
    G, W, V, steps = 3, 4, eos + 3, 7        # (ids behind the table's are never allowed)
    search = BeamSearch(_ctx(), G, W, steps, eos=(eos,))
    state = torch.full((G * W,), fsm.state, dtype=torch.int32, device="cuda")
    states = BeamStates([(state, 0)], W)
    print(f"[case] beams under a grammar G={G} W={W} V={V}", flush=True)
    while not search.finished():
        x = rng.normal(0, 2, (G * W, V)).astype(np.float32)
        x[:, [V - 1, 4]] += 6.0
        bits = fsm.dfa.mask(table, state, V)
        allow = unpacked(bits, V)
        check(rows_at(x, "f32", 1, 1), beams(rng, G, W), empty_pool(G, W), W, (eos,), allow=allow, bits=bits, what="grammar")
        x[~allow] = np.nan
        search.step(torch.from_numpy(x).cuda(), bits)
        beam_reorder(_ctx(), states, search.parents)
        now = state.cpu().numpy()
        for r, t in enumerate(search.tokens.view(-1).tolist()):
            if t >= 0:
                now[r], viable = fsm.dfa.advance(table, int(now[r]), t)
                assert viable, (r, t)
        state.copy_(torch.from_numpy(now))
    ended = 0
    for g, hyps in enumerate(search.sequences()):
        assert hyps
        for h in hyps:
            ids = h.tokens[:-1] if h.finished else h.tokens
            s = fsm.state
            for t in ids:
                s, viable = fsm.dfa.advance(table, s, t)
                assert viable
            if h.finished:
                ended += 1
                assert h.tokens[-1] == eos and re.fullmatch(PATTERN, b"".join(tokens[t] for t in ids).decode())
    assert ended
