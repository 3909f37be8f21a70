"""BeamDecoder where a GreedyDecoder was: the same arguments, and the same record of a call's times."""
import pytest

from golden_util import load_case
from test_beam_decode_gpu import prompts

pytestmark = pytest.mark.gpu


def test_arguments_and_times(dev):
    from simlingo_amd.decode import BeamDecoder, GreedyDecoder
    from simlingo_amd.engine import VLAEngine
    cfg, P, ex, _ = load_case("leftpad")
    eng = VLAEngine(cfg, dev, P)
    prefix = prompts(cfg, P, ex, eng)[0][0]
    for graph in (True, False):
        kw = dict(max_len=512, max_new_tokens=6, eos_id=-1, use_graph=graph, check_every=2)
        greedy, beam = GreedyDecoder(eng, **kw), BeamDecoder(eng, num_beams=3, **kw)
        for dec in (greedy, beam):
            assert dec.generate(prefix).numel() == 6
        assert beam.last_timing.keys() == greedy.last_timing.keys()
        assert beam.last_timing["decode_steps"] == greedy.last_timing["decode_steps"] == 5
        assert beam.last_timing["prefill_ms"] > 0 and beam.last_timing["decode_ms"] > 0
        ids, _ = beam.search(prefix)
        eos = int(ids[0, 1])
        short = BeamDecoder(eng, num_beams=1, **{**kw, "eos_id": eos, "check_every": 1})
        assert short.generate(prefix)[-1] == eos and short.last_timing["decode_steps"] < 5
