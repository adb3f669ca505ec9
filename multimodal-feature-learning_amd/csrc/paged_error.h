// The error text shared by the two sources behind include/paged_cache.h.
#ifndef MFL_PAGED_ERROR_H
#define MFL_PAGED_ERROR_H

// sets mfl_paged_last_error()'s text (printf format) for this thread; returns false
__attribute__((format(printf, 1, 2))) bool mfl_paged_error(const char* fmt, ...);

#endif
