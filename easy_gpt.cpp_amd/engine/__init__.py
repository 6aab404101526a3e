from .context import GroupTables, StepContext
from .drafting import PromptLookup
from .engine import DTYPES, DraftEntry, Engine, StepEntry, load_model

__all__ = ["DTYPES", "DraftEntry", "Engine", "GroupTables", "PromptLookup", "StepContext", "StepEntry", "load_model"]
