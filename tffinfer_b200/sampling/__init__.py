from .params import SamplingParams, GREEDY, RANDOM, TOP_K, TOP_P
from .controls import LogitControls, mask_of
from .sampler import Sampler, uniform_for
