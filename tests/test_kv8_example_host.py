"""The serving example's requests without a GPU, with a plain loop in the place of the pages' kernels."""
import random

import pytest

from tests.test_gpu_pages import plain_cut, plain_take


@pytest.mark.parametrize("sequences,pages,prompt,tokens,chunk", [(1, 9, 100, 40, 32), (2, 10, 100, 40, 16), (5, 12, 120, 60, 32), (8, 30, 200, 100, 256), (3, 100, 50, 50, 8)])
def test_every_request_is_finished(sequences, pages, prompt, tokens, chunk):
    """With pages for little more than one request most are put off now and then: none is lost or cut short, and somebody always gets on."""
    from amdgpu_rustdsl_b200.kv8_example import Requests
    rng, made, page, room = random.Random(sequences), [], 16, prompt + tokens

    def new():
        n = rng.randint(1, prompt)
        made.append([n, n + rng.randint(1, tokens)])
        return made[-1]

    requests = Requests(sequences, new)
    free, table, lengths = [pages, 0, 0, 0, *range(pages)], [[-1] * -(-room // page) for _ in range(sequences)], [0] * sequences
    last = 0
    for step in range(4000):
        asked = requests.ask(chunk)
        assert max(asked) > 0
        granted = plain_take(free, table, lengths, asked, page, 1)[0]
        before = len(requests.finished)
        over = requests.step(granted)
        for r in requests.finished[before:]:
            assert any(r is x and n == r[1] for x, n in zip(current, lengths)) if step else True
        if over is not None:
            plain_cut(free, table, lengths, [0 if x else room for x in over], page)
        assert requests.lengths == lengths
        current = list(requests.now)
        last = step if len(requests.finished) > before else last
        assert step - last < 3 * sequences * room
    unfinished = {id(r) for r in requests.now}
    assert len(requests.finished) + sequences == len(made) and all((id(r) in unfinished) != any(r is f for f in requests.finished) for r in made)
    # in the order in which they came, but for those that are still under way
    assert len(requests.finished) > 10 and (requests.put_off > 0) == (sequences in (2, 5, 8))


def test_too_few_pages_for_one_request_are_refused(capsys):
    from amdgpu_rustdsl_b200.kv8_example import main
    with pytest.raises(SystemExit):
        main(["--prompt", "100", "--tokens", "100", "--pages", "3"])
    assert "too few for one request" in capsys.readouterr().err
