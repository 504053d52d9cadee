from .step import Engine, StepEntry, StepError, OutOfPages
from .continuations import Accepted, DraftEntry, DraftStep
