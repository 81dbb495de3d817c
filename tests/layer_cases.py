"""
Layers for the tests of grouped_linear's tiles: lengths of the groups, inputs, outputs, elements that every row and weight line is off its
16-byte place by, the nonlinearity, and the tiles that the forward call, the gradient of x and that of the weights take.
"""
from tests.linear_plan import ROWS16, T64, T128, T128D, T256D


def _ragged(groups, mean, step=37):
    """ lengths around `mean`, hardly any of them a multiple of 32, one of 0 and one of 1 """
    lengths = [mean + (step*i) % 61 - 30 for i in range(groups)]
    lengths[1 % groups], lengths[-1] = (0, 1) if groups > 4 else (lengths[1 % groups], lengths[-1])
    return lengths


# name: (lengths, K, N, shift, nonlin, forward, dx, dw, joint)
CASES = {
    'wide': (_ragged(8, 5200, 311), 1000, 1992, 0, None, T256D, T256D, T256D, True),
    'wide, tanh': (_ragged(26, 560), 1544, 1608, 0, 'tanh', T256D, T256D, T256D, True),
    'wide inputs': ([20000, 0, 12761], 768, 200, 0, None, T128D, T256D, T128D, False),
    'wide outputs': ([20000, 0, 12761], 200, 768, 0, 'sigmoid', T256D, T128D, T128D, True),
    'many groups': (_ragged(44, 205), 520, 520, 0, None, T128D, T128D, T256D, False),
    'square': (_ragged(36, 205), 520, 520, 0, 'tanh', T128D, T128D, T128D, True),
    'square, shifted': (_ragged(36, 205), 520, 520, 1, None, T128, T128, T128, True),
    'no multiple of 8': (_ragged(36, 205), 516, 524, 0, 'tanh', T128D, T128, T128, True),
    'small groups': (_ragged(200, 47), 136, 136, 0, None, T64, T64, T128D, False),
    'small groups, odd': (_ragged(200, 47), 131, 133, 1, 'relu', T64, T64, T128, False),
    'one group': ([25001], 136, 136, 0, None, T128D, T128D, T64, False),
    'one group, shifted': ([25001], 136, 136, 1, 'sigmoid', T128, T128, T64, False),
    'one group, narrow': ([25001], 60, 72, 0, None, T128D, T64, T64, True),
    'handfuls': (_ragged(300, 31), 40, 72, 0, None, T64, T64, T64, True),
    'few rows': ([7, 0, 20, 1, 9]*12, 200, 264, 0, 'tanh', ROWS16, ROWS16, T128D, False),
}
